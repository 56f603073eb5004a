"""Beam selection over logits of all sizes: every kind of row decides by itself, in rows of one chunk per run and of several."""

import pytest
import torch

from axonn_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCORES = (-0.25, -0.6213, -1.0337, -1.4519)      # no two differ by a step of 16-bit logits: equal values are equal for a reason
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _same(logits, scores):
    want = ops.beam_select(logits, scores)
    got = ops.beam_select(logits.to(DEV), scores.to(DEV))
    for name in ("tokens", "parents"):
        wrong = (getattr(got, name).cpu() != getattr(want, name)).any(1)
        assert not bool(wrong.any()), f"{name} of prompts {wrong.nonzero().flatten().tolist()[:8]}: {getattr(got, name).cpu()[wrong][0]} for {getattr(want, name)[wrong][0]}"
    # one rounding to 32 bits; sums of non-negative terms, each lane's of at most 24 and then of 32 lanes, terms off by at most 2^-22
    # (exp2) and 2^-24 x 12 (a rounded exponent, weighed with its term): (24 + 5 + 4 + 12) 2^-24 < 2^-18 of the sum, its logarithm's error
    finite = want.scores.isfinite()
    assert torch.equal(got.scores.cpu()[~finite], want.scores[~finite])
    assert bool(((got.scores.cpu() - want.scores).abs()[finite] <= 2.0 ** -23 * want.scores[finite].abs() + 2.0 ** -18).all())


def _rows(V, dtype):
    """Rows of ``V`` values, many chunks of 4 KB."""
    g = torch.Generator().manual_seed(V)
    normal = lambda: torch.randn(V, generator=g) * 2  # noqa: E731
    chunk = 4096 // torch.empty(0, dtype=dtype).element_size()
    up = torch.linspace(-3e4, 3e4, V)
    rows = [up, up.flip(0), up * 0.01, torch.zeros(V), normal() * 1e-6, normal() * 500, normal() + 4090, normal() - 4100]
    if dtype != torch.float16:
        rows += [up * 1e30, up.flip(0) * 1e30, torch.full((V,), -3e38), torch.full((V,), 3e38), normal() * 1e7, normal() * 1e37]
        rows += [normal() * 4 + c for c in (1e5, 1e6, 1e7, 3e7, 1e8, 1e10, -1e5, -1e7, -1e10, -1e30)]
    low = [-60000.0, -1e4, -5000.0] if dtype == torch.float16 else [-5000.0, -1e4, -1e9, -1e10, -1e20, -1e30, -3e38]
    for value in low:                            # banned tokens: the first chunk, the last ones, all but one chunk, all but one token
        for keep in (slice(chunk, V), slice(0, V - 2 * chunk), slice(2 * chunk, 3 * chunk), slice(V // 2, V // 2 + 1)):
            row = torch.full((V,), value)
            row[keep] = normal()[keep]
            rows.append(row)
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_all_sizes_each_by_itself(dtype):
    """Every beam of a prompt has the same row, so that all that is selected comes from it."""
    rows = _rows(9001, dtype)
    _same(rows[:, None].expand(-1, 4, -1).contiguous(), torch.tensor(SCORES).expand(len(rows), 4).contiguous())
    _same(rows[:, None].contiguous(), torch.zeros(len(rows), 1))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_all_sizes_beside_ordinary_ones(dtype):
    """The best of the row and the best of an ordinary one 0.37 apart: both are selected, and their sums are compared."""
    rows = _rows(9001, dtype)
    other = (torch.randn(len(rows), 9001, generator=torch.Generator().manual_seed(1)) * 3).to(dtype)
    best, best_other = (x.double().log_softmax(-1).amax(-1) for x in (rows, other))
    scores = torch.stack([torch.zeros(len(rows), dtype=torch.float64), best - best_other - 0.37], 1).float()
    _same(torch.stack([rows, other], 1), scores)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_all_sizes_in_runs_of_several_chunks(dtype):
    """So many rows that a warp takes several chunks of one: masked chunks first, in between and last in a run."""
    chunk = 4096 // torch.empty(0, dtype=dtype).element_size()
    g = torch.Generator().manual_seed(0)
    V, B, K = 8 * chunk, 400, 4
    logits = torch.randn(B * K, 8, chunk, generator=g) * 2
    low = [-60000.0, -1e4] if dtype == torch.float16 else [-1e4, -1e9, -1e10, -1e20, -1e30, -3e38]
    value = torch.tensor(low)[torch.randint(0, len(low), (B * K, 1, 1), generator=g)]
    masked = torch.rand(B * K, 8, generator=g) < 0.6
    masked[:, 0] = torch.arange(B * K) % 2 == 0
    masked[:, 7] &= masked[:, :7].sum(1) < 7             # something is left of every row
    logits = torch.where(masked[..., None], value, logits).to(dtype).view(B, K, V)
    _same(logits, torch.tensor(SCORES).expand(B, K).contiguous())
