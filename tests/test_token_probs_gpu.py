"""The kernels of ``token_log_probs`` against the 64-bit form on the CPU."""

import pytest
import torch

from axonn_b200 import ops
from axonn_b200.ops import _lib

from _vocabulary import check_gradient, check_told, told, told_gradient

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _case(shape, dtype, seed=0, ignored=0.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = (3 * torch.randn(shape, generator=g, device=DEV)).to(dtype)
    tokens = torch.randint(0, shape[-1], shape[:-1], generator=g, device=DEV)
    tokens[torch.rand(shape[:-1], generator=g, device=DEV) < ignored] = -100
    return logits, tokens


def _check(logits, tokens=None, top=0, temperature=1.0, entropy=True, gradient=True, ignore_index=-100):
    z = logits.detach().requires_grad_(gradient)
    before = _lib.launch_count
    got = ops.token_log_probs(z, tokens, entropy=entropy, top=top, temperature=temperature, ignore_index=ignore_index)
    assert _lib.launch_count > before
    want = told(z, tokens, top, temperature, ignore_index)
    check_told(got, want, z.shape[-1], top)
    if not gradient:
        return got
    g = torch.Generator(device=DEV).manual_seed(1)
    kept = z.detach().clone()
    for which in ([0, 1, 2], [0], [1], [2]):
        outs = {i: got[i] for i in which if got[i] is not None}
        if not outs:
            continue
        d = {i: torch.randn(t.shape, generator=g, device=DEV) for i, t in outs.items()}
        (grad,) = torch.autograd.grad(list(outs.values()), z, list(d.values()), retain_graph=True)
        assert grad.dtype == z.dtype and grad.shape == z.shape
        want_d, size = told_gradient(z, tokens, d.get(0), d.get(1), d.get(2), temperature, ignore_index)
        check_gradient(grad, want_d, size, z.shape[-1], want["log_p"])
    assert torch.equal(z.detach().isnan(), kept.isnan()) and torch.equal(z.detach().nan_to_num(), kept.nan_to_num())
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,top,temperature", [
    ((1,), 1, 1.0), ((1, 1), 1, 1.0), ((3, 2), 2, 0.7), ((5, 7), 0, 1.0), ((2, 3, 31), 31, 1.3), ((9, 255), 5, 1.0), ((4, 257), 32, 1.0),
    ((2, 2, 3, 1000), 8, 0.5), ((301, 2048), 3, 1.0), ((7, 2049), 20, 1.0), ((3, 8191), 32, 1.0), ((40, 16385), 1, 2.0), ((2, 32000), 5, 1.0),
    ((5, 50304), 0, 1.0), ((1, 128256), 20, 0.8), ((2, 100003), 7, 1.0), ((700, 301), 4, 1.0)])
def test_told(shape, top, temperature, dtype):
    """One value to many blocks per row, odd vocabularies, one row to more than fit at once; 16-bit logits have many equal values."""
    _check(*_case(shape, dtype, ignored=0.2 if len(shape) > 1 else 0.0), top, temperature)


@pytest.mark.parametrize("entropy,top,tokens", [(False, 0, True), (True, 0, True), (False, 4, True), (True, 4, False), (False, 4, False), (True, 0, False)])
@pytest.mark.parametrize("rows,V", [(3, 4099), (400, 1000)])
def test_what_is_asked_for(entropy, top, tokens, rows, V):
    logits, t = _case((rows, V), torch.bfloat16)
    got = _check(logits, t if tokens else None, top, entropy=entropy)
    assert (got.log_probs is None) == (not tokens) and (got.entropy is None) == (not entropy) and (got.top_tokens is None) == (top == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [64, 333, 4104])
def test_strides(V, dtype):
    """All positions but the last, rows with gaps, off 16 bytes, turned, stretched; tokens that are a slice."""
    logits, tokens = _case((3, 6, V), dtype)
    _check(logits[:, :-1], tokens[:, 1:], 3)
    _check(logits[:, 1::2], tokens[:, ::2], 2)
    _check(logits[..., 1:], tokens.clamp(max=V - 2), 2)
    _check(logits[..., 5:V - 3], tokens.clamp(max=V - 9), 2)
    _check(logits.transpose(0, 1), tokens.t(), 2)
    turned = logits.transpose(1, 2).contiguous().transpose(1, 2)
    _check(turned, tokens, 2)
    _check(logits[:1].expand(4, 6, V), tokens[0].expand(4, 6), 2, gradient=False)
    _check(logits[0, 0].expand(3, 6, V), tokens, 2, gradient=False)
    flat = torch.empty(18 * V + 1, dtype=dtype, device=DEV)
    flat[1:] = logits.reshape(-1)
    _check(flat[1:].view(3, 6, V), tokens, 3)
    four = logits.view(3, 2, 3, V)[:, :, :-1]
    _check(four, tokens.view(3, 2, 3)[:, :, 1:], 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [9, 1030, 40000])
def test_masks_and_values_that_are_no_numbers(V, dtype):
    low = torch.finfo(dtype).min
    logits, tokens = _case((16, V), dtype, ignored=0.0)
    logits[0] = -INF
    logits[1, 3] = NAN
    logits[2, V - 1] = INF
    logits[3], logits[3, V // 2] = -INF, 1.0
    tokens[3] = V // 2
    logits[4] = low
    logits[5, ::2] = low
    logits[6, 1::2] = -INF
    logits[7, :-2] = -INF                                  # fewer tokens than alternatives
    logits[8] = -INF
    logits[8, ::3] = low                                   # -inf beside the lowest value
    logits[9] = 0.0
    logits[9, ::2] = -0.0                                  # equal values
    logits[10] = INF
    logits[11] = NAN
    logits[12, 0], logits[12, V - 1] = -NAN, NAN
    logits[13], logits[13, 2] = -INF, NAN
    logits[14] = torch.finfo(dtype).max
    logits[15, 1], logits[15, 2] = torch.finfo(dtype).max, low
    tokens[7], tokens[8] = 0, 1
    got = _check(logits, tokens, min(9, V))
    assert got.log_probs[3] == 0 and got.entropy[3] == 0
    assert got.top_tokens[9].tolist() == list(range(min(9, V)))
    _check(logits, tokens, min(9, V), temperature=0.3)
    tokens[::2] = -100
    _check(logits, tokens, min(9, V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 200])
def test_order_of_the_vocabulary(rows, dtype):
    """Rows that grow, that fall, that have few different values, and large ones: the bounds and references of what has been read move."""
    V = 50000
    up = torch.linspace(-60, 60, V, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    kinds = [up, up.flip(0), up * 1e-3, (torch.randn(V, generator=g, device=DEV) * 2).round(), up * (500 if dtype == torch.float16 else 5e36),
             torch.where(torch.arange(V, device=DEV) < 49990, 1.0, 2.0), torch.full((V,), -7.0, device=DEV)]
    logits = torch.stack(kinds).repeat(-(-rows // len(kinds)), 1)[:max(rows, len(kinds))].to(dtype)
    tokens = torch.randint(0, V, logits.shape[:1], generator=g, device=DEV)
    if rows == 1:
        for i in range(len(kinds)):
            _check(logits[i:i + 1], tokens[i:i + 1], 32)
    else:
        _check(logits, tokens, 32, gradient=False)
        _check(logits[:7], tokens[:7], 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 129), (1, 33000), (4, 128256), (900, 2600), (300, 9001)])
def test_few_values_above_the_others(rows, V, dtype):
    """Masks that leave fewer tokens than alternatives, or these in a few places; rows of one value but for some, and what grows behind that."""
    j = torch.arange(V, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn(V, generator=g, device=DEV)
    kinds = [torch.where(torch.rand(V, generator=g, device=DEV) < 0.9999, -INF, x), torch.where(j % 1024 < 16, x, -INF), torch.where(j % 256 == 9, x, -INF),
             torch.where(j >= V - 7, x, -INF), torch.where(j % 511 == 0, 1.0, 0.0), torch.where(j % 97 == 96, -1.0, 0.0), torch.where(j < V // 2, 2.0, j / V * 4),
             torch.where(j < V - 40, -x.abs(), 5.0), torch.where(j % 8 == 7, 3.0, j / V), torch.where(j < 3, 3.0, -INF), j / V * 8 + x / 16]
    some = torch.stack(kinds).repeat(-(-rows // len(kinds)), 1)[:max(rows, len(kinds))].to(dtype)
    tokens = some.float().argmax(-1)
    for top in (1, 5, 20, 32):
        if rows == 1:
            for i in range(len(kinds)):
                _check(some[i:i + 1], tokens[i:i + 1], top, gradient=False)
        else:
            _check(some, tokens, top, gradient=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [65, 4097, 70000])
def test_magnitudes_that_count_as_zero(V, dtype):
    """Below 2^-126 they are all equal, so that the first of them come first."""
    small = torch.tensor(2.0 ** -130, device=DEV)
    j = torch.arange(V, device=DEV)
    kinds = [(-small).expand(V), torch.where(j < V // 2, 0.0, small), torch.where(j % 2 == 0, -small, small), torch.where(j % 50 == 3, -small, -1.0),
             torch.where(j % 3 == 0, -small, -INF), torch.where(j == V - 1, small, -small), torch.where(j % 2 == 0, -small, torch.tensor(-2.0 ** -126, device=DEV))]
    logits = torch.stack(kinds).to(dtype)
    want = torch.where(logits.float().abs() < 2.0 ** -126, 0.0, logits.float()).to(dtype)
    tokens = torch.zeros(len(kinds), dtype=torch.int64, device=DEV)
    for top in (1, 20):
        check_told(ops.token_log_probs(logits, tokens, entropy=True, top=top), told(want, tokens, top), V, top)


def test_tokens_outside_the_vocabulary():
    logits, _ = _case((5, 77), torch.bfloat16)
    tokens = torch.tensor([77, -1, -100, 76, 1 << 40], device=DEV)
    got = _check(logits, tokens, 2)
    assert got.log_probs.isnan().tolist() == [True, True, False, False, True]
    _check(logits, tokens.clamp(0, 76), 2, ignore_index=76)


def test_all_rows_are_ignored():
    logits, tokens = _case((6, 500), torch.float32, ignored=2.0)
    got = _check(logits, tokens, 3)
    assert got.log_probs.eq(0).all() and got.top_tokens.eq(-1).all()


def test_same_bits_every_time_and_on_another_stream():
    logits, tokens = _case((600, 5003), torch.bfloat16)
    logits.requires_grad_()

    def both():
        r = ops.token_log_probs(logits, tokens, entropy=True, top=6, temperature=0.9)
        return [*r, *torch.autograd.grad([r.log_probs, r.entropy], logits, [torch.ones_like(r.log_probs), torch.ones_like(r.entropy)])]

    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(both(), want))


@pytest.mark.parametrize("rows,V", [(2, 30001), (500, 1024)])
def test_captured_into_graphs(rows, V):
    """Two graphs, forward and backward, replayed in turn on new values."""
    logits, tokens = _case((rows, V), torch.bfloat16)
    logits.requires_grad_()
    d = torch.randn(rows, device=DEV)

    def both():
        r = ops.token_log_probs(logits, tokens, entropy=True, top=5)
        return [*r, *torch.autograd.grad([r.log_probs, r.entropy], logits, [d, d])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(both())
    for seed in (1, 2):
        new, t = _case((rows, V), torch.bfloat16, seed)
        with torch.no_grad():
            logits.copy_(new)
            tokens.copy_(t)
        want = both()
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_rows_beyond_2_31_values():
    V = 131072
    logits = torch.zeros(16500, V, dtype=torch.bfloat16, device=DEV)
    tokens = torch.full((16500,), -100, device=DEV)
    last, t = _case((3, V), torch.bfloat16, ignored=0.0)
    logits[-3:], tokens[-3:] = last, t
    logits.requires_grad_()
    r = ops.token_log_probs(logits, tokens, entropy=True, top=4)
    want = told(last, t, 4)
    check_told(ops.TokenLogProbs(*(x[-3:] for x in r)), want, V, 4)
    assert r.log_probs[:-3].eq(0).all()
    d = torch.randn(16500, device=DEV)
    (g,) = torch.autograd.grad(r.log_probs, logits, d)
    check_gradient(g[-3:], *told_gradient(last, t, d[-3:]), V, want["log_p"])
    assert g[0].eq(0).all() and g[8000].eq(0).all()


def test_refusals():
    z, t = torch.randn(2, 5, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    for bad in (lambda: ops.token_log_probs(z, t.cpu()), lambda: ops.token_log_probs(z.double(), t), lambda: ops.token_log_probs(z, t, top=6),
                lambda: ops.token_log_probs(z)):
        with pytest.raises(ValueError):
            bad()
    z.requires_grad_()
    r = ops.token_log_probs(z, t)
    with torch.no_grad():
        z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.log_probs.sum().backward()
    r = ops.token_log_probs(z, t)
    (g,) = torch.autograd.grad(r.log_probs.square().sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()
    assert ops.token_log_probs(z[:0], t[:0], entropy=True, top=2).top_tokens.shape == (0, 2)
