"""The block cache's CPU forms against the 64-bit oracles, what its functions refuse, and what their C entries refuse on the host."""

import shutil

import pytest
import torch

from _block_cache import E4M3, INT8, attend64, attend_bound, make_cache, make_tables, rope_table, same_bits, store64
from axonn_b200 import ops
from axonn_b200.ops import _lib

native = pytest.mark.skipif(not (_lib.available() or shutil.which("nvcc")), reason="native library not built")


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_plan_by_hand():
    """Three requests: one with room in its block, one that starts, one whose table is full; then a list that runs out."""
    tables = torch.tensor([[7, -1, -1], [-1, -1, -1], [1, 2, 3]], dtype=torch.int32)
    plan = ops.plan_blocks(_i32(10, 0, 47), _i32(8, 17, 3), tables, _i32(9, 9, 4, 5, 6, 8), _i32(2), 20, 16)
    assert tables.tolist() == [[7, 4, -1], [5, 6, -1], [1, 2, 3]]
    assert plan.lengths.tolist() == [18, 17, 48] and plan.taken.tolist() == [5]
    assert plan.slots[0].tolist() == [7 * 16 + t for t in range(10, 16)] + [64, 65] + [-1] * 12
    assert plan.slots[1].tolist() == [80 + t for t in range(16)] + [96] + [-1] * 3
    assert plan.slots[2].tolist() == [63] + [-1] * 19 and plan.positions[2].tolist() == [47] + [-1] * 19
    assert plan.positions[0, :8].tolist() == list(range(10, 18)) and plan.positions[0, 8:].tolist() == [-1] * 12
    tables = torch.full((3, 2), -1, dtype=torch.int32)
    plan = ops.plan_blocks(_i32(0, 0, 0), _i32(20, 20, 20), tables, _i32(3, 1, 2), _i32(0), 20, 16)
    assert tables.tolist() == [[3, 1], [2, -1], [-1, -1]]
    assert plan.lengths.tolist() == [20, 16, 0] and plan.taken.tolist() == [3] and int((plan.slots >= 0).sum()) == 36
    for R, S in ((0, 3), (2, 0)):
        plan = ops.plan_blocks(_i32(*[5] * R), _i32(*[1] * R), torch.full((R, 2), -1, dtype=torch.int32), _i32(0), _i32(0), S, 16)
        assert plan.slots.shape == (R, S) and plan.lengths.tolist() == [5] * R and plan.taken.tolist() == [0]


@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("first", [0, 5])
def test_store(codes, rope, first):
    torch.manual_seed(first)
    qkv = (torch.randn(2, 30, 2, 4, 32) * 3).bfloat16()
    cache = make_cache(6, 2, 16, 32, codes)
    positions = (first + torch.arange(30))[None].repeat(2, 1).int()
    positions[1, 20:] = -1
    slots = torch.where(positions >= 0, torch.tensor([[0], [48]]) + positions, -1).long()
    table = rope_table(33, 32) if rope else None      # positions 33 and 34 are not in it
    want, q64 = store64(qkv, cache, slots, positions, table)
    layer = ops.BlockLayer(*[t.clone() for t in cache])
    q = ops.store_blocks(qkv, layer, slots, positions, table)
    assert all(same_bits(a, b) for a, b in zip(layer, want))
    if rope:
        assert bool(((q.double() - q64).abs() <= 2.0 ** -8 * q64.abs() + 2.0 ** -21 * qkv.double().abs().max()).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend(dtype):
    lengths, new = [0, 1, 40, 33, 17], [0, 1, 3, 2, 3]
    cache, tables = make_cache(10, 2, 16, 32, E4M3), make_tables(lengths, 3, 16, 10)
    tables[3, 1] = -1
    torch.manual_seed(0)
    q = torch.randn(5, 3, 4, 32).to(dtype)
    out = ops.cached_attention(q, ops.BlockLayer(*cache), tables, _i32(*lengths), _i32(*new))
    want, size = attend64(q, cache, tables, lengths, new)
    assert out.dtype == dtype and bool(((out.double() - want).abs() <= attend_bound(want, size, dtype)).all())


def test_reorder_by_hand():
    """Two groups of three rows: one in the middle of its second block, one on a block border."""
    N, BT = 16, 16
    blocks = ops.BlockLayer(*(t[None] for t in make_cache(N, 1, BT, 16, INT8)))
    before = [t.clone() for t in blocks]
    tables = torch.tensor([[0, 1, -1], [0, 2, -1], [0, 3, -1], [4, 5, 6], [4, 5, 7], [4, 5, 8]], dtype=torch.int32)
    lengths, spare = _i32(20, 20, 20, 32, 32, 32), _i32(9, 10, 11, 12, 13, 14)
    out = ops.reorder_blocks(blocks, tables, lengths, spare, _i32(1, 1, 0, 2, 2, 1).view(2, 3))
    assert out[0].tolist() == [[0, 9, -1], [0, 2, -1], [0, 11, -1], [4, 5, 8], [4, 5, 8], [4, 5, 7]]
    assert out[1].tolist() == lengths.tolist() and out[2].tolist() == [1, 10, 3, 12, 13, 14]
    for t, b in zip(blocks[:2], before[:2]):
        b[0, 9, :, :4], b[0, 11, :, :4] = b[0, 2, :, :4].clone(), b[0, 1, :, :4].clone()
        assert torch.equal(t, b)
    for t, b in zip(blocks[2:], before[2:]):
        b[0, 9], b[0, 11] = b[0, 2].clone(), b[0, 1].clone()
        assert torch.equal(t, b)


def test_select_by_hand():
    inf, nan = float("inf"), float("nan")
    p = torch.tensor([[0.5, 0.25, 0.25], [0.125, 0.125, 0.75]]).log()[None]
    step = ops.beam_select(p, torch.tensor([[0.0, -inf]]))
    assert step.tokens.tolist() == [[0, 1]] and step.parents.tolist() == [[0, 0]] and step.done is None
    step = ops.beam_select(p, torch.tensor([[-1.0, -1.0]]), torch.tensor([[False, False]]), 2)
    assert step.tokens.tolist() == [[2, 0]] and step.parents.tolist() == [[1, 0]] and step.done.tolist() == [[True, False]]
    step = ops.beam_select(p, torch.tensor([[-1.0, -1.25]]), torch.tensor([[True, False]]), 1)
    assert step.tokens.tolist() == [[1, 2]] and step.scores[0, 0] == -1 and step.done.tolist() == [[True, False]]
    p[0, 0, 1] = nan
    step = ops.beam_select(p, torch.zeros(1, 2))
    assert step.parents.tolist() == [[1, 1]] and step.tokens.tolist() == [[2, 0]]
    step = ops.beam_select(p, torch.tensor([[inf, nan]]))
    assert step.parents.tolist() == [[0, 0]] and step.tokens.tolist() == [[0, 1]] and step.scores.tolist() == [[-inf, -inf]]
    assert ops.beam_select(p[:0], torch.zeros(0, 2)).tokens.shape == (0, 2)


def _layer(N=4, G=2, BT=16, D=32, dtype=E4M3):
    return ops.BlockLayer(*make_cache(N, G, BT, D, dtype))


def _refused(error, words, f, *args, **kw):
    with pytest.raises(error, match=words):
        f(*args, **kw)


def test_refusals_of_plan():
    ok = [_i32(3, 4), _i32(1, 1), torch.zeros(2, 3, dtype=torch.int32), _i32(1, 2), _i32(0), 1, 16]
    ops.plan_blocks(*ok)
    for at, value in ((0, ok[0].long()), (0, ok[2]), (1, _i32(1)), (2, ok[2][:1]), (2, torch.zeros(3, 2, dtype=torch.int32).T), (2, _i32(1)),
                      (2, torch.zeros(2, 0, dtype=torch.int32)), (3, _i32()), (3, ok[3].float()), (4, _i32(0, 0)), (5, -1), (6, 17), (6, 256)):
        _refused(ValueError, None, ops.plan_blocks, *[value if i == at else a for i, a in enumerate(ok)])
    _refused(ValueError, "tensors on", ops.plan_blocks, *[ok[0], ok[1].to("meta"), *ok[2:]])


def test_refusals_of_store():
    layer, qkv, slots = _layer(), torch.randn(1, 3, 2, 4, 32), torch.arange(3)[None]
    positions, table = slots.int(), rope_table(16, 32)
    ops.store_blocks(qkv, layer, slots, positions, table)
    f = ops.store_blocks
    for bad in (qkv[0], qkv[:, :, :1], qkv[:, :, :, :1], qkv[..., :16]):
        _refused(ValueError, "qkv", f, bad, layer, slots)
    for bad in (slots.int(), slots[:, :2], torch.zeros(3, 1, dtype=torch.int64).T[:, ::2]):
        _refused(ValueError, "slots", f, qkv, layer, bad)
    _refused(ValueError, "positions", f, qkv, layer, slots, None, table)
    _refused(ValueError, "positions", f, qkv, layer, slots, slots, table)
    for bad in (table.double(), table[:, :8], table[..., 0]):
        _refused(ValueError, "rope table", f, qkv, layer, slots, positions, bad)
    _refused(RuntimeError, "no derivative", f, qkv.clone().requires_grad_(), layer, slots)
    with torch.no_grad():
        f(qkv.clone().requires_grad_(), layer, slots)
    _refused(TypeError, "codes", f, qkv, layer._replace(k=layer.k.float()), slots)
    _refused(TypeError, "codes", f, qkv, layer._replace(v=layer.v.view(torch.int8)), slots)
    _refused(TypeError, "scales", f, qkv, layer._replace(k_scale=layer.k_scale.double()), slots)
    _refused(ValueError, "scales", f, qkv, layer._replace(v_scale=layer.v_scale[:3]), slots)
    _refused(ValueError, "dense", f, qkv, layer._replace(k=layer.k.transpose(0, 1).contiguous().transpose(0, 1)), slots)
    _refused(ValueError, "blocks hold", f, qkv, ops.BlockLayer(*make_cache(4, 2, 8, 32, INT8)), slots)


def test_refusals_of_attention():
    layer, q, tables, lengths = _layer(), torch.randn(2, 1, 4, 32), torch.zeros(2, 3, dtype=torch.int32), _i32(3, 4)
    f = ops.cached_attention
    f(q, layer, tables, lengths)
    for bad in (q[0], q[:, :, :3], q[..., :16], q[:, :, None, :2]):
        _refused(ValueError, "q must be", f, bad, layer, tables, lengths)
    for bad in (tables.long(), tables[:1], tables[0]):
        _refused(ValueError, "tables", f, q, layer, bad, lengths)
    _refused(ValueError, "lengths", f, q, layer, tables, lengths.long())
    _refused(ValueError, "new", f, q, layer, tables, lengths, _i32(1))
    for bad in (float("nan"), float("inf")):
        _refused(ValueError, "scale", f, q, layer, tables, lengths, None, bad)
    _refused(RuntimeError, "no derivative", f, q.clone().requires_grad_(), layer, tables, lengths)
    assert f(q[:0], layer, tables[:0], lengths[:0]).shape == (0, 1, 4, 32)
    assert not bool(f(q, layer, tables[:, :0], lengths).any())


def test_refusals_of_reorder():
    blocks = ops.BlockLayer(*(t[None] for t in _layer()))
    tables, rows, parents = torch.zeros(4, 2, dtype=torch.int32), _i32(0, 0, 0, 0), torch.zeros(2, 2, dtype=torch.int32)
    f = ops.reorder_blocks
    f(blocks, tables, rows, rows, parents)
    _refused(ValueError, None, f, _layer(), tables, rows, rows, parents)
    _refused(ValueError, "parents", f, blocks, tables, rows, rows, parents[:1])
    _refused(ValueError, "parents", f, blocks, tables, rows, rows, parents.long())
    _refused(ValueError, "reorder_blocks takes", f, blocks, tables, rows, rows, parents[0])
    _refused(ValueError, "lengths", f, blocks, tables, rows[:3], rows, parents)
    _refused(ValueError, "spare", f, blocks, tables, rows, rows.long(), parents)


def test_refusals_of_select():
    x, s, d = torch.zeros(2, 3, 5), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.bool)
    f = ops.beam_select
    f(x, s, d, 4)
    for bad in (x[0], x.double(), x[..., :0], x.long()):
        _refused(ValueError, "logits", f, bad, s)
    _refused(ValueError, "beams", f, torch.zeros(1, 33, 5), torch.zeros(1, 33))
    _refused(ValueError, "beams", f, torch.zeros(1, 0, 5), torch.zeros(1, 0))
    for bad in (s.double(), s[:1], s[0]):
        _refused(ValueError, "scores", f, x, bad)
    _refused(ValueError, "together", f, x, s, d)
    _refused(ValueError, "together", f, x, s, None, 3)
    _refused(ValueError, "done", f, x, s, d.int(), 3)
    for bad in (-1, 5):
        _refused(ValueError, "eos_id", f, x, s, d, bad)
    _refused(RuntimeError, "no derivative", f, x.clone().requires_grad_(), s)


@native
def test_refusals_of_the_c_entries():
    """On the host, before anything is launched: addresses that are never used."""
    L, p = _lib.lib(), 4096
    error = lambda: L.axb_last_error().decode()  # noqa: E731
    assert L.axb_plan_blocks(*[p] * 9, 1, 1, 1, 1, 48, None) == -1 and "16, 32, 64 or 128" in error()
    assert L.axb_plan_blocks(*[p] * 9, 1, 0, 1, 1, 16, None) == -1 and "empty" in error()
    store = lambda q=p, stride=64, D=64, BT=16, dtype=0: L.axb_store_blocks(  # noqa: E731
        q, 64, stride, 64, p, p, p, p, p, p, p, p, 1, 1, 1, 1, D, 1, BT, 1, dtype, 0, None)
    attend = lambda q=p, stride=64, D=64, BT=16, dtype=0, work=p: L.axb_cached_attention(  # noqa: E731
        q, 64, stride, 64, p, p, p, p, p, p, None, p, work, 1, 1, 1, 1, D, 1, 1, BT, 1.0, dtype, 0, None)
    for call in (store, attend):
        assert call(q=p + 8) == -1 and "aligned" in error()
        assert call(stride=60) == -1 and "stride" in error()
        assert call(D=96) == -1 and "64 or 128" in error()
        assert call(BT=24) == -1 and "16, 32, 64 or 128" in error()
        assert call(dtype=2) == -1 and "bf16 or fp16" in error()
    assert attend(work=p + 4) == -1 and "aligned" in error()
    reorder = lambda k=p, R=4, K=2, row=64, L_=1: L.axb_reorder_blocks(k, p, p, p, p, p, p, p, p, p, p, L_, R, K, 1, 1, 1, 16, row, None)  # noqa: E731
    assert reorder(k=p + 8) == -1 and "aligned" in error()
    assert reorder(R=5) == -1 and "empty" in error()
    assert reorder(row=40) == -1 and "16" in error()
    assert reorder(L_=70000) == -1 and "65535" in error()
    select = lambda K=2, V=4, dtype=0, work=p: L.axb_beam_select(p, p, None, -1, p, p, p, None, work, 1, K, V, dtype, None)  # noqa: E731
    assert select(K=33) == -1 and "beams" in error()
    assert select(V=(1 << 30) + 1) == -1 and "vocabulary" in error()
    assert select(dtype=3) == -1 and "logits" in error()
    assert select(work=p + 4) == -1 and "aligned" in error()


@pytest.mark.parametrize("taken,got", [(-3, 2), (0, 2), (3, 1), (4, 0), (9, 0), (2**31 - 1, 0)])
def test_plan_from_any_number_of_taken_blocks(taken, got):
    """Nothing outside the list is named."""
    tables = torch.full((1, 4), -1, dtype=torch.int32)
    one = lambda x: torch.tensor([x], dtype=torch.int32)  # noqa: E731
    free = torch.tensor([10, 11, 12, 13], dtype=torch.int32)
    plan = ops.plan_blocks(one(0), one(20), tables, free, one(taken), 20, 16)
    first = min(max(taken, 0), 4)
    assert tables[0].tolist() == [10 + first + i if i < got else -1 for i in range(4)]
    assert int(plan.lengths) == min(20, 16 * got) and int(plan.taken) == first + got


def test_plan_refuses_tables_of_more_tokens_than_lengths_count():
    none = torch.empty(0, dtype=torch.int32)
    with pytest.raises(ValueError, match="2.31"):
        ops.plan_blocks(none, none, torch.empty(0, 1 << 27, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                        torch.zeros(1, dtype=torch.int32), 1, 16)
    L, p = _lib.lib(), 4096
    assert L.axb_plan_blocks(*[p] * 9, 1, 1, 1 << 27, 1, 16, None) == -1 and "2^31" in L.axb_last_error().decode()
