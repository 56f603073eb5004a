"""Steps in which no row has a new token with a place, and caches that are full, on the CPU."""

import pytest
import torch

from _block_cache import E4M3, INT8, make_cache, rope_table, same_bits
from _dist import run_distributed
from axonn_b200 import ops


@pytest.mark.parametrize("P", [0, 1, 3])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_a_step_that_stores_nothing(P, rope, codes):
    cache = make_cache(4, 2, 16, 64, codes)
    layer = ops.BlockLayer(*(t.clone() for t in cache))
    slots, positions = torch.full((3, 5), -1, dtype=torch.int64), torch.full((3, 5), -1, dtype=torch.int32)
    q = ops.store_blocks(torch.randn(3, 5, 2, P + 2, 64).bfloat16(), layer, slots, positions, rope_table(40, 64) if rope else None)
    assert all(same_bits(a, b) for a, b in zip(layer, cache))
    if rope:
        assert q.shape == (3, 5, 2 * P, 64) and q.dtype == torch.bfloat16 and not bool(q.any())
    else:
        assert q is None


def _full(rank, world):
    from axonn_b200 import axonn as ax
    from axonn_b200.models import BlockCache, Llama, LlamaConfig

    ax.init(G_inter=1, G_data=1, G_intra_r=1, G_intra_c=1, G_intra_d=1)
    torch.manual_seed(0)
    model = Llama(LlamaConfig(n_layers=1, hidden=64, n_heads=4, n_kv_heads=2, ffn=128, vocab=96, seq_len=40), dtype=torch.float32).eval()
    with torch.no_grad():
        cache = BlockCache(model, 2, 16, 16)
        cache.plan(16)
        model(torch.zeros(2, 16, dtype=torch.long), cache=cache)
        cache.plan(1)
        assert cache.new.tolist() == [0, 0] and cache.lengths.tolist() == [16, 16]
        assert bool(model(torch.zeros(2, 1, dtype=torch.long), cache=cache).isfinite().all())


def test_a_model_whose_cache_is_full():
    run_distributed(_full, 1)
