"""Queries of attention over the block cache whose values differ by many octaves within a row."""

import pytest
import torch

from _block_cache import E4M3, INT8, attend64, attend_bound, make_cache, make_tables
from axonn_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("S,heads", [(1, 4), (4, 4), (17, 8)])
@pytest.mark.parametrize("codes,dtype,D,small", [(E4M3, torch.bfloat16, 128, -26), (INT8, torch.bfloat16, 64, -28), (INT8, torch.float16, 64, -13)])
def test_small_values_beside_a_large_one(S, heads, codes, dtype, D, small):
    """One value of a row is 2^-small times the others' size, and every key is zero there: the scores are those of the small values."""
    lengths, BT = [300, 33, 20], 32
    blocks = sum(-(-n // BT) for n in lengths)
    k, v, ks, vs = make_cache(blocks, 1, BT, D, codes)
    k = k.float()
    k[..., 5] = 0
    k, ks = k.to(codes), torch.full_like(ks, 2.0 ** (-6 - small))
    tables = make_tables(lengths, -(-300 // BT), BT, blocks)
    q = torch.randn(len(lengths), S, heads, D, generator=torch.Generator().manual_seed(D))
    q = (q.clamp(-3, 3) * 2.0 ** small)
    q[..., 5] = 1.0
    q = q.to(dtype)
    out = ops.cached_attention(q.to(DEV), ops.BlockLayer(*(t.to(DEV) for t in (k, v, ks, vs))), tables.to(DEV),
                               torch.tensor(lengths, dtype=torch.int32, device=DEV)).cpu()
    want, size = attend64(q, (k, v, ks, vs), tables, lengths)
    # fp16 holds what is scaled by 2^14 to multiples of 2^-24: most values exactly; the others move scores by what they are off times keys
    off = (q.double() * 2.0 ** 14 - (q.float() * 2.0 ** 14).half().double()).abs() * 2.0 ** -14
    for r, n in enumerate(lengths):
        token = torch.arange(n)
        keys = k.float()[tables[r].long()[token // BT], 0, token % BT].abs().double() * 2.0 ** (-6 - small)
        moved = (off[r] @ keys.T).amax(-1, keepdim=True) * D ** -0.5
        bound = attend_bound(want[r], size[r], dtype) + torch.expm1(2 * moved) * size[r]
        assert bool(((out[r].double() - want[r]).abs() <= bound).all())
        assert float(moved.max()) < 2.0 ** -9
