"""Calls of the vocabulary's operators, and of the layers and functions on them, at the ends of what they take: on the CPU."""

import pytest
import torch

from _dist import run_distributed


def _grid(world, depth=1):
    from axonn_b200 import axonn as ax

    ax.init(G_inter=1, G_data=world // depth, G_intra_r=1, G_intra_c=1, G_intra_d=depth)


def _rows_outside(rank, world):
    """A device whose lookups look at no index (on a GPU torch's ends the program) is never asked for rows that the table has not got."""
    from axonn_b200.intra_layer import Embedding

    _grid(world)
    for scale in (1.0, 2.0):
        layer = Embedding(40, 8, expert_mode=True, scale=scale)
        there = layer.rows(23, 17, "cpu")
        for device in ("cpu", "meta"):
            layer = layer.to(device)
            for grad in (False, True):
                with torch.set_grad_enabled(grad):
                    for first, count in ((24, 17), (-1, 2), (40, 1), (1 << 40, 3)):
                        with pytest.raises(IndexError):
                            layer.rows(first, count, device)
                    assert layer.rows(23, 17, device).shape == (17, 8) and layer.rows(0, 40, device).shape == (40, 8)
                    for first in (0, 40, 50):
                        assert layer.rows(first, 0, device).shape == (0, 8)
    assert there.shape == (17, 8)


def test_rows_that_the_table_has_not_got():
    run_distributed(_rows_outside, 1)
