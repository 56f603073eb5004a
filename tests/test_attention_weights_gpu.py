"""Attention over the block cache where one token has nearly all of the weight: what the weak rest adds up to is kept."""

import math

import pytest
import torch

from _block_cache import E4M3, INT8, as_codes, attend64, attend_bound, make_tables
from axonn_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _sink(lengths, gaps, S, D, BT, codes, at=0):
    """One KV head, a query head for each of ``gaps``: the token ``at`` has a score of ``gap`` (of the natural exponent) and values of zero,
    all others scores from -0.4 to 0.4 and values of some size."""
    g = torch.Generator().manual_seed(len(lengths) + D)
    blocks = sum(-(-n // BT) for n in lengths)
    tables = make_tables(lengths, -(-max(lengths) // BT), BT, blocks)
    k, v = torch.zeros(blocks, 1, BT, D), 40 + 60 * torch.rand(blocks, 1, BT, D, generator=g)
    k[..., 1] = torch.randint(-6, 7, (blocks, 1, BT), generator=g).float()
    for r, n in enumerate(lengths):
        b, t = int(tables[r, min(at, n - 1) // BT]), min(at, n - 1) % BT
        k[b, 0, t, 0], k[b, 0, t, 1], v[b, 0, t] = 64.0, 0.0, 0.0
    q = torch.zeros(len(lengths), S, len(gaps), D)
    q[..., 0], q[..., 1] = torch.tensor(gaps), 4.0
    one = torch.full((blocks, 1), 2.0 ** -6)             # values of the codes 64: ones
    return q, (as_codes(k, codes), as_codes(v, codes), one, one.clone()), tables


@pytest.mark.parametrize("codes,dtype,D,BT", [(E4M3, torch.bfloat16, 128, 64), (INT8, torch.float16, 64, 16)])
@pytest.mark.parametrize("S,heads", [(1, 4), (4, 4), (8, 2), (16, 4), (17, 8)])
@pytest.mark.parametrize("lengths", [[32, 20, 160], [3000, 700], [40000]])
@pytest.mark.parametrize("at", [0, 130])
def test_a_token_with_nearly_all_of_the_weight(S, heads, lengths, at, codes, dtype, D, BT):
    """Weights down to e^-18 = 2^-26 of the largest one keep the precision of every other, 2^-11 of them; what lies below would lose at
    most 2^-37 of the largest weight for each token.  Scores are sums of two products: the bound's share for them is not used up."""
    gaps = [18.0, 16.0, 14.0, 10.0, 17.0, 15.0, 12.0, 6.0][:heads]
    q, cache, tables = _sink(lengths, gaps, S, D, BT, codes, at)
    q = q.to(dtype)
    out = ops.cached_attention(q.to(DEV), ops.BlockLayer(*(t.to(DEV) for t in cache)), tables.to(DEV),
                               torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=1.0).cpu()
    want, size = attend64(q, cache, tables, lengths, scale=1.0)
    lost = torch.tensor(lengths, dtype=torch.float64)[:, None, None, None] * 2.0 ** -37 * 100 * 2.0 ** -6
    assert bool(((out.double() - want).abs() <= attend_bound(want, size, dtype) + lost + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all())
    seen = want.abs().amax((2, 3)) > 0
    assert bool((out.abs().amax((2, 3))[seen] > 0).all())


@pytest.mark.parametrize("S", [1, 8, 33])
def test_weights_that_rise_along_the_sequence(S):
    """Every token weighs twice as much as the one before: references are raised all along, by a little each time, and no weight
    becomes infinite.  D 64, scores up to 0.69 x 200."""
    lengths, BT, D = [200, 90, 1], 16, 64
    blocks = sum(-(-n // BT) for n in lengths)
    tables = make_tables(lengths, 13, BT, blocks)
    k, v = torch.zeros(blocks, 1, BT, D), torch.randn(blocks, 1, BT, D, generator=torch.Generator().manual_seed(0)) * 64
    for r, n in enumerate(lengths):
        for t in range(n):
            k[int(tables[r, t // BT]), 0, t % BT, :2] = torch.tensor([float(t // 16), float(t % 16)])
    one = torch.ones(blocks, 1)
    cache = (as_codes(k, INT8), as_codes(v, E4M3).float().round().clamp(-127, 127).to(torch.int8), one, one)
    q = torch.zeros(len(lengths), S, 4, D)
    q[..., 0], q[..., 1] = 16.0, 1.0
    q = q.half()
    scale = math.log(2.0)
    out = ops.cached_attention(q.to(DEV), ops.BlockLayer(*(t.to(DEV) for t in cache)), tables.to(DEV),
                               torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=scale).cpu()
    want, size = attend64(q, cache, tables, lengths, scale=scale)
    # scores of up to 200 in octaves, exact but for their product with the scale: 200 x 2^-23, which moves weights by 0.7 of that
    bound = attend_bound(want, size, torch.float16) + 200 * 2.0 ** -23 * (size + want.abs())
    assert bool(((out.double() - want).abs() <= bound).all())
