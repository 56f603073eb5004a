"""The block cache's kernels against 64-bit oracles (``_block_cache.py``) and, where results are exact, to the bit."""

import os
import subprocess
import sys

import pytest
import torch

from _block_cache import E4M3, INT8, attend64, attend_bound, make_cache, make_tables, put, rope_table, same_bits, store64
from axonn_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gpu(*ts):
    return [t.to(DEV) if torch.is_tensor(t) else t for t in ts]


# ----------------------------------------------------------------------------- plan

@pytest.mark.parametrize("R,S,BT,W,N,taken", [(1, 1, 16, 1, 1, 0), (5, 1, 16, 3, 40, 7), (300, 1, 64, 9, 500, 0), (700, 3, 16, 5, 4000, 13),
                                              (7, 2500, 64, 60, 400, 1), (3, 1025, 128, 20, 9, 0), (2000, 2, 32, 4, 900, 5),
                                              (257, 1, 16, 4, 3, 3), (4, 100, 16, 3, 50, 60)])
def test_plan(R, S, BT, W, N, taken):
    """The same as the CPU form to the last integer: prefix sums over blocks of the grid, full tables, a list that runs out."""
    g = torch.Generator().manual_seed(R + S)
    lengths = torch.randint(0, W * BT + 1, (R,), generator=g).int()
    lengths[::3] = (lengths[::3] // BT) * BT
    new = torch.randint(-1, S + 2, (R,), generator=g).int()
    free = torch.randperm(N, generator=g).int()
    tables = make_tables([0] * R, W, BT, 1)
    for r in range(R):
        tables[r, :-(-int(lengths[r]) // BT)] = 10000 + r
    taken = torch.tensor([taken], dtype=torch.int32)
    here = tables.to(DEV)
    got = ops.plan_blocks(*_gpu(lengths, new), here, *_gpu(free, taken), S, BT)
    want = ops.plan_blocks(lengths, new, tables, free, taken, S, BT)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and torch.equal(here.cpu(), tables)


# ----------------------------------------------------------------------------- store

def _store_case(R, S, G, P, D, BT, codes, dtype, context, seed=0):
    g = torch.Generator().manual_seed(seed)
    before = [(context * (r + 1)) // R for r in range(R)]
    new = [S - (r * S) // (2 * R) for r in range(R)]
    W = -(-(context + S) // BT)
    blocks = sum(-(-(b + n) // BT) for b, n in zip(before, new)) + 2
    tables = make_tables([b + n for b, n in zip(before, new)], W, BT, blocks, seed)
    slots, positions = torch.full((R, S), -1, dtype=torch.int64), torch.full((R, S), -1, dtype=torch.int32)
    for r in range(R):
        for i in range(new[r]):
            at = before[r] + i
            slots[r, i], positions[r, i] = int(tables[r, at // BT]) * BT + at % BT, at
    qkv = (torch.randn(R, S, G, P + 2, D, generator=g) * torch.exp2(torch.randint(-3, 4, (R, 1, G, P + 2, 1), generator=g).float())).to(dtype)
    return qkv, make_cache(blocks, G, BT, D, codes, seed), slots, positions, rope_table(W * BT, D)


@pytest.mark.parametrize("R,S,G,P,D,BT,codes,dtype,context", [
    (3, 1, 2, 4, 128, 64, E4M3, torch.bfloat16, 100), (5, 1, 1, 1, 64, 16, INT8, torch.float16, 47), (2, 1, 3, 2, 128, 16, INT8, torch.bfloat16, 0),
    (2, 16, 2, 1, 128, 64, E4M3, torch.float16, 77), (2, 33, 2, 3, 64, 32, E4M3, torch.bfloat16, 90), (3, 130, 1, 1, 128, 128, INT8, torch.bfloat16, 5),
    (1, 200, 2, 1, 128, 32, E4M3, torch.bfloat16, 0), (2, 300, 1, 2, 64, 128, INT8, torch.float16, 200), (4, 7, 2, 8, 64, 16, E4M3, torch.bfloat16, 31)])
@pytest.mark.parametrize("rope", [False, True])
def test_store(R, S, G, P, D, BT, codes, dtype, context, rope):
    """Codes and scales to the bit (powers of two, one rounding each); queries are rounded once (half a step; 32-bit products before)."""
    qkv, cache, slots, positions, table = _store_case(R, S, G, P, D, BT, codes, dtype, context)
    table = table if rope else None
    want, q64 = store64(qkv, cache, slots, positions, table)
    layer = ops.BlockLayer(*_gpu(*cache))
    q = ops.store_blocks(qkv.to(DEV), layer, slots.to(DEV), positions.to(DEV), None if table is None else table.to(DEV))
    for a, b in zip(layer, want):
        assert same_bits(a.cpu(), b)
    cpu = ops.BlockLayer(*[t.clone() for t in cache])
    q_cpu = ops.store_blocks(qkv, cpu, slots, positions, table)
    assert all(same_bits(a, b) for a, b in zip(cpu, want))
    if rope:
        wide = qkv.double().abs().amax(-1)[:, :, :, :-2].reshape(R, S, -1, 1)
        assert bool(((q.cpu().double() - q64).abs() <= torch.finfo(dtype).eps / 2 * q64.abs() + 2.0 ** -22 * wide + 2.0 ** -25).all())
        assert torch.equal(q.cpu(), q_cpu)
    else:
        assert q is None


@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_store_of_infinities_nan_zeros_and_tiny_values(codes):
    """Infinities are the largest code, NaN is NaN (0 in int8), the scale is that of the finite values; a head of zeros has the least
    scale, values below its reach are zeros."""
    inf, nan = float("inf"), float("nan")
    qkv = torch.zeros(4, 1, 2, 3, 64)
    qkv[0, 0, 0, 1, :5] = torch.tensor([1.0, inf, -inf, nan, -2.0])
    qkv[1, 0, 0, 1, :3] = torch.tensor([nan, inf, -inf])
    qkv[2, 0, 0, 2, :2] = torch.tensor([3e38, -1e-38])
    qkv[3, 0, 1, 1, :2] = torch.tensor([1e-39, 2.0 ** -120])
    qkv = qkv.bfloat16()
    cache = make_cache(4, 2, 16, 64, codes)
    slots = torch.arange(4)[:, None] * 16
    layer, cpu = ops.BlockLayer(*_gpu(*cache)), ops.BlockLayer(*[t.clone() for t in cache])
    ops.store_blocks(qkv.to(DEV), layer, slots.to(DEV))
    ops.store_blocks(qkv, cpu, slots)
    for a, b in zip(layer, cpu):
        assert torch.equal(a.cpu().float().nan_to_num(9e9), b.float().nan_to_num(9e9))
    row = layer.k[0, 0, 0, :5].float().cpu()
    most = 448.0 if codes == E4M3 else 127.0
    assert float(layer.k_scale[0, 0]) == (2.0 ** -7 if codes == E4M3 else 2.0 ** -5) and row[1] == most and row[2] == -most
    assert bool(row[3].isnan()) if codes == E4M3 else row[3] == 0
    assert float(layer.k_scale[1, 0]) == 2.0 ** -100 and float(layer.k_scale[3, 1]) == 2.0 ** -100
    assert not bool(layer.k[3, 1, 0].float().any())


def test_store_token_by_token_is_the_store_of_all_but_for_rounding_again():
    """A block filled one token at a time ends with the scale of the whole block; e4m3 codes lose nothing by a power of two but where
    they fall below the least normal code: the difference is at most one step there, 2^-9 of a code."""
    torch.manual_seed(0)
    qkv = (torch.randn(1, 40, 2, 3, 128) * torch.logspace(-1, 1, 40)[None, :, None, None, None]).bfloat16()
    once, steps = (ops.BlockLayer(*_gpu(*make_cache(1, 2, 64, 128, E4M3))) for _ in range(2))
    slots = torch.arange(40, device=DEV)[None]
    ops.store_blocks(qkv.to(DEV), once, slots)
    for i in range(40):
        ops.store_blocks(qkv[:, i:i + 1].to(DEV), steps, slots[:, i:i + 1].contiguous())
    assert torch.equal(once.k_scale, steps.k_scale) and torch.equal(once.v_scale, steps.v_scale)
    for a, b in ((once.k, steps.k), (once.v, steps.v)):
        assert float((a[:, :, :40].float() - b[:, :, :40].float()).abs().max()) <= 2.0 ** -9


def test_store_of_strided_and_unaligned_projections():
    """A slice of a wider projection (its strides are read as they are) and one that starts off 16 bytes (copied)."""
    qkv, cache, slots, positions, table = _store_case(2, 5, 2, 2, 64, 16, E4M3, torch.bfloat16, 20)
    want = ops.BlockLayer(*_gpu(*cache))
    q_want = ops.store_blocks(qkv.to(DEV), want, slots.to(DEV), positions.to(DEV), table.to(DEV))
    wide = torch.randn(2, 5, 3, 4, 64).bfloat16().to(DEV)
    wide[:, :, 1:] = qkv.to(DEV)
    off = torch.empty(qkv.numel() + 1, dtype=qkv.dtype, device=DEV)[1:].view(qkv.shape).copy_(qkv)
    heads_apart = torch.empty(2, 5, 2, 4, 128, dtype=qkv.dtype, device=DEV)[..., :64].copy_(qkv)
    for other in (wide[:, :, 1:], off, heads_apart):
        layer = ops.BlockLayer(*_gpu(*cache))
        q = ops.store_blocks(other, layer, slots.to(DEV), positions.to(DEV), table.to(DEV))
        assert torch.equal(q, q_want) and all(same_bits(a, b) for a, b in zip(layer, want))


# ----------------------------------------------------------------------------- attend

def _attend(q, cache, tables, lengths, new=None, **kw):
    """Runs the kernel and compares; returns the result."""
    out = ops.cached_attention(q.to(DEV), ops.BlockLayer(*_gpu(*cache)), tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV),
                               None if new is None else torch.tensor(new, dtype=torch.int32, device=DEV), **kw).cpu()
    want, size = attend64(q, cache, tables, lengths, new, **kw)
    far = (out.double() - want).abs() - attend_bound(want, size, q.dtype)
    assert float(far.max()) <= 2.0 ** -24 and bool(out.isfinite().all())
    return out


@pytest.mark.parametrize("G,P,D", [(1, 1, 64), (2, 4, 128), (1, 8, 64), (2, 3, 128), (1, 12, 128), (4, 1, 128), (1, 20, 64)])
@pytest.mark.parametrize("BT,codes,dtype", [(16, E4M3, torch.bfloat16), (64, E4M3, torch.float16), (128, INT8, torch.bfloat16), (32, INT8, torch.float16)])
def test_attend_one_token(G, P, D, BT, codes, dtype):
    """Lengths of none, one, tile and block borders, several blocks."""
    lengths = [0, 1, 15, 16, 17, BT, BT + 1, 2 * BT, 3 * BT - 1, 0, 5 * BT]
    W = 5
    blocks = sum(-(-n // BT) for n in lengths) + 3
    torch.manual_seed(G * P)
    q = torch.randn(len(lengths), 1, G * P, D).to(dtype)
    out = _attend(q, make_cache(blocks, G, BT, D, codes), make_tables(lengths, W, BT, blocks), lengths)
    assert not bool(out[0].any()) and not bool(out[9].any())


@pytest.mark.parametrize("S,P,D,codes", [(2, 1, 64, E4M3), (3, 4, 128, INT8), (8, 1, 128, E4M3), (8, 2, 64, INT8), (17, 1, 64, E4M3), (40, 3, 128, E4M3)])
def test_attend_several_tokens(S, P, D, codes):
    """Queries see up to their own token; ragged numbers of new ones, none, more than the sequence has; queries behind are zeros."""
    lengths = [S, S + 1, 50, 70, 5, 33, 0]
    new = [S, S, max(S - 1, 1), 0, 5 if S >= 5 else S, 1, 0]
    BT, W = 32, 5
    torch.manual_seed(S)
    q = torch.randn(len(lengths), S, 2 * P, D).bfloat16()
    cache, tables = make_cache(40, 2, BT, D, codes), make_tables(lengths, W, BT, 40)
    out = _attend(q, cache, tables, lengths, new)
    for r, m in enumerate(new):
        assert not bool(out[r, m:].any())
    _attend(q, cache, tables, [max(n, S) for n in lengths[:3]] + [70, 40, 40, 40], None) if S <= 33 else None


def test_attend_long_sequences_are_split():
    """Sequences of many warps, of every position of the cuts, beside short ones and none."""
    lengths = [4001, 3, 0, 2500, 16, 1, 3999]
    torch.manual_seed(0)
    q = torch.randn(len(lengths), 1, 8, 128).bfloat16()
    blocks = sum(-(-n // 64) for n in lengths)
    _attend(q, make_cache(blocks, 2, 64, 128, E4M3), make_tables(lengths, 63, 64, blocks), lengths)


def test_attend_more_requests_than_one_launch_counts():
    torch.manual_seed(0)
    R = 4100
    lengths = [(7 * r) % 19 for r in range(R)]
    blocks = sum(-(-n // 16) for n in lengths)
    q = torch.randn(R, 1, 1, 64).half()
    _attend(q, make_cache(blocks, 1, 16, 64, INT8), make_tables(lengths, 2, 16, blocks), lengths)


def test_attend_blocks_of_very_different_scales():
    """Scales of values from 2^-46 to 2^34, one of a block of zeros: the result is as exact as its largest terms.  (Sums of p |v| are the
    bound's measure, and large blocks with small weights belong to them.)"""
    BT, lengths = 16, [160, 64]
    k, v, ks, vs = make_cache(14, 1, BT, 64, E4M3)
    vs = torch.exp2(torch.tensor([-46.0, 34, -6, -100, 0, 20, -20, 3, -30, 10, -6, -6, 7, -11]))[:, None]
    v[3] = torch.zeros(1, BT, 64).to(E4M3)
    torch.manual_seed(2)
    _attend(torch.randn(2, 1, 2, 64).bfloat16(), (k, v, ks, vs), make_tables(lengths, 10, BT, 14), lengths)
    # a block of huge values that the softmax gives next to nothing: scores far below the others'
    k = torch.zeros(2, 1, 16, 64)
    k[0], k[1, :, :, 0] = 0, -1
    v = torch.randn(2, 1, 16, 64) * 64
    cache = as_layer(k * 64, v, torch.full((2, 1), 2.0 ** -6), torch.tensor([[2.0 ** -6], [2.0 ** 24]]))
    q = torch.zeros(1, 1, 1, 64)
    q[..., 0] = 160.0
    tables = torch.tensor([[0, 1]], dtype=torch.int32)
    out = ops.cached_attention(q.bfloat16().to(DEV), ops.BlockLayer(*_gpu(*cache)), tables.to(DEV), torch.tensor([32], dtype=torch.int32, device=DEV))
    want, size = attend64(q.bfloat16(), cache, tables, [32])
    assert bool(((out.cpu().double() - want).abs() <= attend_bound(want, size, torch.bfloat16)).all()) and float(want.abs().max()) < 2


def as_layer(k, v, ks, vs):
    return k.to(E4M3), v.to(E4M3), ks, vs


@pytest.mark.parametrize("poison", [0x7f, 0xff])
def test_what_is_masked_may_be_nan(poison):
    """NaN codes behind a sequence, in blocks of nobody, and NaN scales of those; a stored NaN that some queries see and others do not
    reaches the queries that see it and no others."""
    BT, lengths, S = 16, [5, 20, 40, 31], 4
    cache = make_cache(12, 2, BT, 64, E4M3)
    tables = make_tables(lengths, 3, BT, 12)
    used = torch.zeros(12, BT, dtype=torch.bool)
    for r, n in enumerate(lengths):
        for t in range(n):
            used[int(tables[r, t // BT]), t % BT] = True
    torch.manual_seed(1)
    q = torch.randn(4, S, 4, 64).bfloat16()
    want = _attend(q, cache, tables, lengths)
    bad = [t.clone() for t in cache]
    for c in bad[:2]:
        c.view(torch.uint8).transpose(1, 2)[~used] = poison
    for s in bad[2:]:
        s[~used.any(1)] = float("nan")
    layer = ops.BlockLayer(*_gpu(*bad))
    args = (q.to(DEV), layer, tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    assert torch.equal(ops.cached_attention(*args).cpu(), want)
    for which in (0, 1):      # key, value of token 18 of the second request: queries 0 and 1 (tokens 16, 17) do not see it
        b, t = int(tables[1, 1]), 2
        worse = [x.clone() for x in bad]
        worse[which].view(torch.uint8)[b, 1, t, 7] = poison
        out = ops.cached_attention(args[0], ops.BlockLayer(*_gpu(*worse)), *args[2:]).cpu()
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[1, 2:, 2:, :] = True if which == 0 else (torch.arange(64) == 7)
        assert torch.equal(out[~hit], want[~hit]) and bool(out[hit].isnan().all())


def test_attend_tables_that_lack_blocks():
    """-1 and ids outside the cache within a sequence count as absent tokens, all of them as an empty sequence."""
    lengths = [60, 40, 33]
    cache, tables = make_cache(12, 1, 16, 128, INT8), make_tables(lengths, 4, 16, 12)
    tables[0, 1], tables[0, 3], tables[1, :] = -1, 12, -1
    torch.manual_seed(1)
    out = _attend(torch.randn(3, 1, 2, 128).bfloat16(), cache, tables, lengths)
    assert not bool(out[1].any())
    _attend(torch.randn(3, 1, 2, 128).bfloat16(), cache, tables, [60, 40, 1000])      # longer than its table: what there is of it


@pytest.mark.parametrize("scale", [0.0, -0.07, 0.5])
def test_attend_scales(scale):
    torch.manual_seed(1)
    lengths = [40, 3]
    q = torch.randn(2, 1, 4, 64).half() * 0.25
    _attend(q, make_cache(4, 2, 16, 64, E4M3), make_tables(lengths, 3, 16, 4), lengths, scale=scale)


def test_attend_queries_of_all_sizes():
    """Queries are scaled by a power of two into fp16: rows of large and of small values, of zeros, a row with large and small ones."""
    torch.manual_seed(1)
    q = torch.randn(5, 1, 2, 128)
    factor = torch.tensor([2.0 ** 60, 2.0 ** -60, 0.0, 1.0, 1.0])
    q = (q * factor[:, None, None, None]).bfloat16()
    q[4, ..., 1:] *= 2.0 ** -18
    lengths = [30, 30, 30, 1, 30]
    k, v, ks, vs = make_cache(10, 1, 16, 128, E4M3)
    ks = ks.clone()
    tables = make_tables(lengths, 2, 16, 10)
    ks[tables[0].long()] *= 2.0 ** -60
    ks[tables[1].long()] *= 2.0 ** 60
    _attend(q, (k, v, ks, vs), tables, lengths)


def test_attend_strides():
    """Queries as the view of a packed projection, transposed, a slice, off 16 bytes."""
    torch.manual_seed(1)
    lengths, new = [40, 33], [3, 2]
    cache, tables = make_cache(6, 2, 16, 64, E4M3), make_tables(lengths, 3, 16, 6)
    qkv = torch.randn(2, 3, 2, 5, 64).bfloat16()
    q = qkv[:, :, :, :3]
    want = _attend(q.reshape(2, 3, 6, 64), cache, tables, lengths, new)
    layer = ops.BlockLayer(*_gpu(*cache))
    rest = (layer, tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), torch.tensor(new, dtype=torch.int32, device=DEV))
    there = q.reshape(2, 3, 6, 64).to(DEV)
    off = torch.empty(there.numel() + 1, dtype=there.dtype, device=DEV)[1:].view(there.shape).copy_(there)
    for other in (qkv.to(DEV)[:, :, :, :3], there.transpose(0, 1).contiguous().transpose(0, 1), there.transpose(1, 2).contiguous().transpose(1, 2),
                  torch.cat([there, there], -1)[..., :64], off):
        assert torch.equal(ops.cached_attention(other, *rest).cpu(), want)


# ----------------------------------------------------------------------------- reorder

@pytest.mark.parametrize("L,B,K,W,BT,G,D,codes", [(1, 1, 2, 1, 16, 1, 64, E4M3), (3, 2, 4, 3, 32, 2, 128, INT8), (2, 5, 3, 4, 64, 5, 64, E4M3),
                                                  (2, 1, 8, 2, 128, 40, 32, INT8)])
def test_reorder(L, B, K, W, BT, G, D, codes):
    """To the bit against the CPU form: parents that are others', one's own, repeated, outside the group; lengths on block borders and
    full tables."""
    R, g = B * K, torch.Generator().manual_seed(L + K)
    N = R * (W + 1) + 1
    parents = torch.randint(-1, K + 1, (B, K), generator=g).int()
    length = torch.randint(0, W * BT + 1, (B,), generator=g)
    length[0] = (W - 1) * BT + 5
    lengths = length.repeat_interleave(K).int()
    ids = torch.randperm(N, generator=g).int()
    tables, spare = ids[:R * W].view(R, W).contiguous(), ids[R * W:R * W + R].contiguous()
    caches = [make_cache(N, G, BT, D, codes, seed=i) for i in range(L)]
    blocks = ops.BlockLayer(*(torch.stack([c.view(torch.uint8) if c.element_size() == 1 else c for c in cs]).view(cs[0].dtype) for cs in zip(*caches)))
    here = ops.BlockLayer(*_gpu(*blocks))
    got = ops.reorder_blocks(here, *_gpu(tables, lengths, spare, parents))
    want = ops.reorder_blocks(blocks, tables, lengths, spare, parents)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and all(same_bits(a.cpu(), b) for a, b in zip(here, blocks))


# ----------------------------------------------------------------------------- together

def _steps(beams, device, streams=None):
    """Prompts of two requests, then tokens one at a time with reordering of beams: plan, store, attend, reorder as they are used."""
    G, P, D, BT, W, S0 = 2, 2, 64, 16, 6, 30
    R = 2 * beams
    g = torch.Generator().manual_seed(3)
    N = R * (W + 2)
    ids = torch.randperm(N, generator=g).int()
    spare, free = ids[:R].to(device), ids[R:].contiguous().to(device)
    layers = [ops.BlockLayer(*(t.to(device) for t in make_cache(N, G, BT, D, E4M3))) for _ in range(1)]
    stacked = ops.BlockLayer(*(t.unsqueeze(0) for t in layers[0]))
    layer = ops.BlockLayer(*(t[0] for t in stacked))
    tables = torch.full((R, W), -1, dtype=torch.int32, device=device)
    lengths, taken = torch.zeros(R, dtype=torch.int32, device=device), torch.zeros(1, dtype=torch.int32, device=device)
    table = rope_table(W * BT, D).to(device)
    outs = []
    for step in range(12):
        S = S0 if step == 0 else 1
        new = torch.tensor([S0 - 7 * (r // beams) if step == 0 else 1 for r in range(R)], dtype=torch.int32, device=device)
        qkv = torch.randn(R, S, G, P + 2, D, generator=g).bfloat16().to(device)
        plan = ops.plan_blocks(lengths, new, tables, free, taken, S, BT)
        q = ops.store_blocks(qkv, layer, plan.slots, plan.positions, table)
        outs.append(ops.cached_attention(q, layer, tables, plan.lengths, new))
        lengths, taken = plan.lengths, plan.taken
        if beams > 1:
            parents = torch.randint(0, beams, (2, beams), generator=g).int().to(device)
            tables, lengths, spare = ops.reorder_blocks(stacked, tables, lengths, spare, parents)
    return outs, tables, lengths, spare, stacked


@pytest.mark.parametrize("beams", [1, 3])
def test_a_run_of_all_of_them(beams):
    """Generation's calls in turn on the GPU and on the CPU: the same tables and cache to the bit, outputs within two roundings to bf16
    (one each) and the bound of the attention's probabilities, for which sums of p |v| of up to four stand."""
    got, want = _steps(beams, DEV), _steps(beams, "cpu")
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got[1:4], want[1:4])) and all(same_bits(a.cpu(), b) for a, b in zip(got[4], want[4]))
    for a, b in zip(got[0], want[0]):
        assert bool(((a.cpu().float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 4 * (2.0 ** -11 + 2.0 ** -13)).all())


def test_a_captured_step_replays():
    """A step of decoding in a graph: new inputs in the same places, the state advanced in place; two graphs replayed on two streams at
    once do not disturb each other."""
    G, P, D, BT, W, R = 2, 4, 128, 32, 4, 3
    torch.manual_seed(0)

    def state(seed):
        layer = ops.BlockLayer(*_gpu(*make_cache(R * W, G, BT, D, INT8, seed)))
        return dict(layer=layer, tables=torch.full((R, W), -1, dtype=torch.int32, device=DEV), lengths=torch.zeros(R, dtype=torch.int32, device=DEV),
                    taken=torch.zeros(1, dtype=torch.int32, device=DEV), free=torch.arange(R * W, dtype=torch.int32, device=DEV),
                    new=torch.ones(R, dtype=torch.int32, device=DEV), qkv=torch.zeros(R, 1, G, P + 2, D, dtype=torch.bfloat16, device=DEV),
                    table=rope_table(W * BT, D).to(DEV))

    def step(s):
        p = ops.plan_blocks(s["lengths"], s["new"], s["tables"], s["free"], s["taken"], 1, BT)
        q = ops.store_blocks(s["qkv"], s["layer"], p.slots, p.positions, s["table"])
        out = ops.cached_attention(q, s["layer"], s["tables"], p.lengths)
        s["lengths"].copy_(p.lengths)
        s["taken"].copy_(p.taken)
        return out
    inputs = torch.randn(60, R, 1, G, P + 2, D, dtype=torch.bfloat16, device=DEV)
    eager, want = state(0), []
    for x in inputs:
        eager["qkv"].copy_(x)
        want.append(step(eager).clone())
    step(state(0))                                          # warm up
    states, graphs, outs, streams = [state(0), state(0)], [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(s))
        graphs.append(graph)
    torch.cuda.synchronize()
    got = [[], []]
    for x in inputs:
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                states[i]["qkv"].copy_(x)
                graphs[i].replay()
                got[i].append(outs[i].clone())
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want)) and torch.equal(states[i]["lengths"], eager["lengths"])


def test_attend_on_another_stream_repeats_its_bits():
    torch.manual_seed(0)
    lengths = [2000, 1, 700]
    q = torch.randn(3, 1, 8, 128).bfloat16().to(DEV)
    layer = ops.BlockLayer(*_gpu(*make_cache(44, 2, 64, 128, E4M3)))
    args = (q, layer, make_tables(lengths, 32, 64, 44).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    want = ops.cached_attention(*args)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = [ops.cached_attention(*args) for _ in range(5)]
        torch.cuda.current_stream().synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 codes: the last block, through store and attention."""
    BT, G, D = 128, 4, 128
    N = (1 << 32) // (BT * G * D) + 3
    k, v = (torch.zeros(N, G, BT, D, dtype=torch.int8, device=DEV) for _ in range(2))
    layer = ops.BlockLayer(k, v, torch.ones(N, G, device=DEV), torch.ones(N, G, device=DEV))
    torch.manual_seed(0)
    qkv = torch.randn(1, 20, G, 3, D).bfloat16()
    small = make_cache(1, G, BT, D, INT8)
    slots = torch.arange(20)[None]
    ops.store_blocks(qkv.to(DEV), layer, (slots + (N - 1) * BT).to(DEV))
    want, _ = store64(qkv, small, slots)
    assert torch.equal(layer.k[N - 1, :, :20].cpu(), want[0][0, :, :20]) and torch.equal(layer.v_scale[N - 1].cpu(), want[3][0])
    q = torch.randn(1, 1, G, D).bfloat16()
    out = ops.cached_attention(q.to(DEV), layer, torch.tensor([[N - 1]], dtype=torch.int32, device=DEV), torch.tensor([20], dtype=torch.int32, device=DEV))
    o64, size = attend64(q, want, torch.zeros(1, 1, dtype=torch.int32), [20])
    assert bool(((out.cpu().double() - o64).abs() <= attend_bound(o64, size, q.dtype)).all())


def test_put_writes_single_codes():
    c = torch.zeros(2, 2).to(E4M3)
    put(c, (1, 1), torch.tensor(2.0).to(E4M3))
    assert c.float().tolist() == [[0.0, 0.0], [0.0, 2.0]]


def test_refusals_on_the_gpu():
    """What the kernels lack is refused, not computed otherwise."""
    cache = make_cache(2, 2, 16, 32, E4M3)
    layer = ops.BlockLayer(*_gpu(*cache))
    slots, one = torch.zeros(1, 1, dtype=torch.int64, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="64 or 128"):
        ops.store_blocks(torch.zeros(1, 1, 2, 3, 32, device=DEV).bfloat16(), layer, slots)
    with pytest.raises(ValueError, match="64 or 128"):
        ops.cached_attention(torch.zeros(1, 1, 2, 32, device=DEV).bfloat16(), layer, one[None], one)
    layer = ops.BlockLayer(*_gpu(*make_cache(2, 2, 16, 64, E4M3)))
    with pytest.raises(TypeError, match="bf16 or fp16"):
        ops.store_blocks(torch.zeros(1, 1, 2, 3, 64, device=DEV), layer, slots)
    with pytest.raises(TypeError, match="bf16 or fp16"):
        ops.cached_attention(torch.zeros(1, 1, 2, 64, device=DEV), layer, one[None], one)
    with pytest.raises(ValueError, match="tensors on"):
        ops.cached_attention(torch.zeros(1, 1, 2, 64, device=DEV).half(), layer, one[None].cpu(), one)
    off = torch.empty(layer.k.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(layer.k.shape).view(E4M3)
    with pytest.raises(ValueError, match="16 bytes"):
        ops.store_blocks(torch.zeros(1, 1, 2, 3, 64, device=DEV).half(), layer._replace(k=off), slots)


def test_native_host_paths_launch_the_same(monkeypatch):
    """The calls through the native host paths and through Python: the same bits, the same refusals; what the paths do not take (queries
    off 16 bytes, gaps between heads) goes the general way."""
    from axonn_b200.ops import _lib

    assert _lib.host() is not None
    lengths, new = [40, 33], [3, 2]
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    cache, tables = make_cache(6, 2, 16, 64, E4M3), make_tables(lengths, 3, 16, 6).to(DEV)
    torch.manual_seed(0)
    qkv = torch.randn(2, 3, 2, 5, 64).bfloat16().to(DEV)
    table = rope_table(48, 64).to(DEV)
    logits = torch.randn(2, 3, 1000, device=DEV)
    scores, done = -torch.rand(2, 3, device=DEV), torch.tensor([[True, False, False], [False, False, True]], device=DEV)

    def run():
        out = list(ops.plan_blocks(i32(37, 31), i32(*new), tables, i32(5, 4, 3, 2, 1, 0), i32(1), 3, 16))
        layer = ops.BlockLayer(*_gpu(*cache))
        out += [ops.store_blocks(qkv, layer, out[0], out[1], table), *layer]
        assert ops.store_blocks(qkv, layer, out[0]) is None
        for q in (qkv[:, :, :, :3], qkv[:, :, :, :3].reshape(2, 3, 6, 64), torch.cat([qkv, qkv], 3)[:, :, :, 0:6:2]):
            out += [ops.cached_attention(q, layer, tables, i32(*lengths), i32(*new)), ops.cached_attention(q, layer, tables, i32(*lengths), None, 0.1)]
        stacked = ops.BlockLayer(*(t[None] for t in layer))
        out += [*ops.reorder_blocks(stacked, i32(0, 1, 0, 2).view(2, 2), i32(20, 20), i32(4, 5), i32(1, 0).view(1, 2)), *layer]
        out += [*ops.beam_select(logits, scores)[:3], *ops.beam_select(logits, scores, done, 7)]
        for error, call in ((ValueError, lambda: ops.cached_attention(qkv, layer, tables, i32(1))),
                            (ValueError, lambda: ops.beam_select(logits, scores, done, 1000)),
                            (ValueError, lambda: ops.beam_select(logits, scores, done)),
                            (ValueError, lambda: ops.plan_blocks(i32(1), i32(1), tables, i32(0), i32(0), 1, 16)),
                            (RuntimeError, lambda: ops.beam_select(logits.clone().requires_grad_(), scores)),
                            (ValueError, lambda: ops.store_blocks(qkv, layer, out[0], None, table)),
                            (ValueError, lambda: ops.reorder_blocks(layer, tables, i32(1, 2), i32(1, 2), i32(0, 0).view(1, 2)))):
            with pytest.raises(error):
                call()
        return out
    native = run()
    monkeypatch.setattr(_lib, "_HOST", None)
    plain = run()
    assert len(native) == len(plain) and all(same_bits(a, b) for a, b in zip(native, plain))


@pytest.mark.parametrize("taken", [-7, 3, 5, 6, 2**31 - 1])
def test_plan_from_any_number_of_taken_blocks(taken):
    """As on the CPU, whatever number stands there."""
    def plan(device):
        tables = torch.full((3, 4), -1, dtype=torch.int32, device=device)
        numbers = [torch.tensor(x, dtype=torch.int32, device=device) for x in ([0, 0, 0], [20, 5, 70], [10, 11, 12, 13, 14], [taken])]
        return tables, *ops.plan_blocks(numbers[0], numbers[1], tables, numbers[2], numbers[3], 70, 16)
    for got, want in zip(plan("cuda"), plan("cpu")):
        assert torch.equal(got.cpu(), want)


# ----------------------------------------------------------------------------- more than 48 query columns

@pytest.mark.parametrize("S,G,P,D,codes,dtype", [(24, 2, 3, 128, E4M3, torch.bfloat16), (9, 1, 8, 64, INT8, torch.float16), (33, 2, 4, 128, INT8, torch.bfloat16),
                                                 (9, 3, 8, 64, E4M3, torch.float16), (17, 1, 5, 128, E4M3, torch.float16), (130, 1, 1, 64, E4M3, torch.bfloat16),
                                                 (1, 1, 72, 128, INT8, torch.bfloat16), (64, 1, 2, 128, INT8, torch.float16)])
@pytest.mark.parametrize("BT", [16, 128])
def test_attend_many_columns(S, G, P, D, codes, dtype, BT):
    """Groups of 128 columns and what is left of them, tiles of 128 tokens and their borders, sequences that several blocks share."""
    lengths = [700, 129, 128, S, 0, 1000, 1, 300, 127, 2600]
    new = [S, S, max(S - 3, 1), S, 0, 1, 1, S + 5, 0, S]
    W = -(-2600 // BT)
    blocks = sum(-(-n // BT) for n in lengths) + 1
    torch.manual_seed(S)
    q = torch.randn(len(lengths), S, G * P, D).to(dtype)
    cache, tables = make_cache(blocks, G, BT, D, codes), make_tables(lengths, W, BT, blocks)
    out = _attend(q, cache, tables, lengths, new)
    for r, m in enumerate(new):
        assert not bool(out[r, max(m, 0):].any())
    assert torch.equal(out, _attend(q, cache, tables, lengths, new))
    tables[0, 1], tables[9, 3:2000 // BT] = -1, blocks + 7       # blocks that a table lacks, within a tile and several tiles long
    _attend(q, cache, tables, lengths, new)


@pytest.mark.parametrize("poison", [0x7f, 0xff])
@pytest.mark.parametrize("D,BT", [(64, 16), (128, 64)])
def test_what_many_columns_do_not_see_may_be_nan(poison, D, BT):
    """NaN codes behind a sequence and in blocks of nobody; a stored NaN among the new tokens reaches the queries that see it alone."""
    S, lengths = 20, [130, 20, 260, 31, 900]
    W, blocks = -(-900 // BT), sum(-(-n // BT) for n in lengths) + 2
    cache, tables = make_cache(blocks, 2, BT, D, E4M3), make_tables(lengths, W, BT, blocks)
    used = torch.zeros(blocks, BT, dtype=torch.bool)
    for r, n in enumerate(lengths):
        for t in range(n):
            used[int(tables[r, t // BT]), t % BT] = True
    torch.manual_seed(1)
    q = torch.randn(len(lengths), S, 8, D).bfloat16()
    want = _attend(q, cache, tables, lengths)
    bad = [t.clone() for t in cache]
    for c in bad[:2]:
        c.view(torch.uint8).transpose(1, 2)[~used] = poison
    for s in bad[2:]:
        s[~used.any(1)] = float("nan")
    args = (q.to(DEV), ops.BlockLayer(*_gpu(*bad)), tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    assert torch.equal(ops.cached_attention(*args).cpu(), want)
    for r, token in ((0, 127), (0, 128), (2, 245), (4, 899), (4, 880), (1, 7)):
        for which in (0, 1):
            worse = [x.clone() for x in bad]
            worse[which].view(torch.uint8)[int(tables[r, token // BT]), 1, token % BT, 37] = poison
            out = ops.cached_attention(args[0], ops.BlockLayer(*_gpu(*worse)), *args[2:]).cpu()
            hit = torch.zeros_like(out, dtype=torch.bool)
            hit[r, token - (lengths[r] - S):, 4:, :] = True if which == 0 else (torch.arange(D) == 37)
            assert torch.equal(out[~hit], want[~hit]) and bool(out[hit].isnan().all())


def test_attend_many_columns_and_blocks_of_very_different_scales():
    """Scales of values from 2^-46 to 2^80: weights whose logarithms lie apart from their values'."""
    BT, lengths = 16, [160, 64]
    k, v, ks, vs = make_cache(14, 1, BT, 64, E4M3)
    torch.manual_seed(2)
    q = torch.randn(2, 9, 8, 64).bfloat16()
    for top in (34.0, 80.0):
        vs = torch.exp2(torch.tensor([-46.0, top, -6, -100, 0, 20, -20, 3, -30, 10, -6, -6, 7, -11]))[:, None]
        _attend(q, (k, v, ks, vs), make_tables(lengths, 10, BT, 14), lengths)
    for scale in (0.0, -0.07, 0.5):
        _attend(q, (k, v, ks, torch.ones_like(vs)), make_tables(lengths, 10, BT, 14), lengths, scale=scale)


_CAPTURED_FIRST = """
import torch
from axonn_b200 import ops
torch.manual_seed(0)
layer = ops.BlockLayer(*(torch.randint(0, 100, (40, 1, 64, 64), dtype=torch.int8, device="cuda") for _ in range(2)),
                       *(torch.full((40, 1), 2.0 ** -6, device="cuda") for _ in range(2)))
tables = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
lengths = torch.tensor([1200, 77], dtype=torch.int32, device="cuda")
q = torch.zeros(2, 9, 8, 64, dtype=torch.bfloat16, device="cuda")
graphs, outs = [], []
for _ in range(2):
    graphs.append(torch.cuda.CUDAGraph())
    with torch.cuda.graph(graphs[-1]):
        outs.append(ops.cached_attention(q, layer, tables, lengths))
streams = [torch.cuda.Stream(), torch.cuda.Stream()]
for _ in range(3):
    q.normal_()
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    want = ops.cached_attention(q, layer, tables, lengths)
    assert all(torch.equal(o, want) for o in outs) and bool(want.any())
print("same")
"""


def test_attend_many_columns_captured_first():
    """The process's first call is captured, twice; both graphs replay on two streams at once."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", _CAPTURED_FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


def test_attend_many_columns_of_strided_queries_on_another_stream():
    """Queries as the view of a packed projection, more requests than one launch counts; the same bits every time."""
    torch.manual_seed(1)
    R, S = 1030, 9
    lengths = [(7 * r) % 150 for r in range(R)]
    blocks = sum(-(-n // 16) for n in lengths)
    qkv = torch.randn(R, S, 1, 10, 64).bfloat16()
    cache, tables = make_cache(blocks, 1, 16, 64, INT8), make_tables(lengths, 10, 16, blocks)
    args = (ops.BlockLayer(*_gpu(*cache)), tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    there = qkv.to(DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = [ops.cached_attention(there[:, :, :, :-2], *args) for _ in range(3)]
        torch.cuda.current_stream().synchronize()
    assert all(torch.equal(g, got[0]) for g in got)
    some = [0, 1, 22, 149, 700, 1023, 1024, 1025, 1029]
    want, size = attend64(qkv[some, :, 0, :-2], cache, tables[some], [lengths[r] for r in some])
    assert bool(((got[0][some].cpu().double() - want).abs() <= attend_bound(want, size, torch.bfloat16) + 2.0 ** -24).all())
