"""Planning, storing and attending where tables lack blocks or name ones outside the cache: as on the CPU, to the bit."""

import pytest
import torch

from _block_cache import E4M3, INT8, attend64, attend_bound, make_cache, rope_table, same_bits
from axonn_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _plan_and_store(device, lengths, new, tables, free, S, G, P, D, BT, codes, dtype, rope, blocks):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    tables = tables.clone().to(device)
    plan = ops.plan_blocks(i32(lengths), i32(new), tables, i32(free), i32([0]), S, BT)
    qkv = torch.randn(len(lengths), S, G, P + 2, D, generator=torch.Generator().manual_seed(S)).to(dtype).to(device)
    layer = ops.BlockLayer(*(t.clone().to(device) for t in make_cache(blocks, G, BT, D, codes)))
    q = ops.store_blocks(qkv, layer, plan.slots, plan.positions, rope_table(tables.shape[1] * BT, D).to(device) if rope else None)
    return tables, plan, qkv, layer, q


@pytest.mark.parametrize("codes,dtype,D", [(E4M3, torch.bfloat16, 128), (INT8, torch.float16, 64)])
@pytest.mark.parametrize("BT,S", [(16, 40), (16, 3), (64, 150), (128, 300), (32, 1)])
@pytest.mark.parametrize("rope", [False, True])
def test_a_table_that_lacks_the_unfinished_block(BT, S, rope, codes, dtype, D):
    """Tokens of the lacking block have no place, those behind it do: they are stored and seen."""
    lengths, new = [BT + 5, 2 * BT - 1, BT, 0, 7], [S, S, S, 0, S]
    W, blocks = 2 + -(-(S + 2 * BT) // BT), 64
    tables = torch.full((5, W), -1, dtype=torch.int32)
    tables[0, 0], tables[1, 0], tables[2, 0] = 50, 51, 52
    args = (lengths, new, tables, list(range(40)), S, 2, 2, D, BT, codes, dtype, rope, blocks)
    here, plan, qkv, layer, q = _plan_and_store(DEV, *args)
    want_tables, want_plan, _, want, want_q = _plan_and_store("cpu", *args)
    assert torch.equal(here.cpu(), want_tables) and all(torch.equal(a.cpu(), b) for a, b in zip(plan, want_plan))
    assert all(same_bits(a.cpu(), b) for a, b in zip(layer, want))
    if rope:
        assert torch.equal(q.cpu(), want_q)
    else:
        q = qkv[:, :, :, :-2].reshape(5, S, 4, D)
    after = plan.lengths.tolist()
    n = [b - a for a, b in zip(lengths, after)]
    out = ops.cached_attention(q, layer, here, plan.lengths, torch.tensor(n, dtype=torch.int32, device=DEV)).cpu()
    o64, size = attend64(q.cpu(), want, want_tables, after, n)
    assert bool(((out.double() - o64).abs() <= attend_bound(o64, size, dtype) + 2.0 ** -24).all()) and bool(out.isfinite().all())


@pytest.mark.parametrize("S", [1, 20, 70])
def test_blocks_outside_the_cache(S):
    """Ids that the cache does not have: their tokens are neither stored nor rotated."""
    tables = torch.full((3, 8), -1, dtype=torch.int32)
    args = ([0, 0, 0], [S, S, S], tables, [5, 900, 2, 64, 3, 1 << 30, 7, 8, 9, 10, 11, 12, 13, 14, 15], S, 2, 1, 64, 16, E4M3, torch.bfloat16, True, 64)
    here, plan, _, layer, q = _plan_and_store(DEV, *args)
    want_tables, want_plan, _, want, want_q = _plan_and_store("cpu", *args)
    assert torch.equal(here.cpu(), want_tables) and all(torch.equal(a.cpu(), b) for a, b in zip(plan, want_plan))
    assert all(same_bits(a.cpu(), b) for a, b in zip(layer, want)) and torch.equal(q.cpu(), want_q)
