"""The kernels of ``embedding`` against the 64-bit form."""

import pytest
import torch

from axonn_b200 import ops
from axonn_b200.ops import _lib

from _vocabulary import HALF_STEP, SMALLEST

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _tokens(n, V, kind, g):
    if kind == "same":
        return torch.full((n,), V // 2, device=DEV)
    if kind == "text":                                     # the r-th token in the share 1 / r
        return (V ** torch.rand(n, generator=g, device=DEV, dtype=torch.float64) - 1).long().clamp_(0, V - 1)
    if kind == "order":
        return torch.arange(n, device=DEV) % V
    if kind == "runs":                                     # segments of 1, 2, 3, ... tokens
        r = ((torch.arange(n, device=DEV) * 2).double().sqrt()).long() % V
        return r[torch.randperm(n, generator=g, device=DEV)]
    return torch.randint(0, V, (n,), generator=g, device=DEV)


def _sums(tokens, dy, V, scale, padding=None):
    """(64-bit gradient, sum of the sizes of its terms, number of terms)."""
    t = tokens.reshape(-1).long()
    d = dy.reshape(-1, dy.shape[-1]).double()
    there = (t >= 0) & (t < V)
    if padding is not None:
        there &= t != padding
    t, d = t[there], d[there]
    zero = torch.zeros(V, d.shape[1], dtype=torch.float64, device=DEV)
    return (zero.index_add(0, t, d, alpha=scale), zero.index_add(0, t, d.abs(), alpha=abs(scale)),
            torch.bincount(t, minlength=V).double()[:, None])


def _check(tokens, weight, dy, scale=1.0, padding=None):
    V, H = weight.shape
    scale = torch.tensor(scale, dtype=torch.float32).item()                                 # the factor is a 32-bit number
    w = weight.detach().requires_grad_()
    before = _lib.launch_count
    out = ops.embedding(tokens, w, scale, padding)
    assert _lib.launch_count > before or out.numel() == 0
    assert out.shape == (*tokens.shape, H) and out.dtype == w.dtype
    want = weight.detach()[tokens.long()].double() * scale
    tol = HALF_STEP[w.dtype] * want.abs() * (1 + 2.0 ** -12) + SMALLEST[w.dtype]            # 32-bit product, then its own type's rounding
    assert scale == 1.0 and torch.equal(out, weight.detach()[tokens.long()]) or bool(((out.double() - want).abs() <= tol).all())
    with torch.no_grad():
        assert torch.equal(ops.embedding(tokens, w, scale, padding), out.detach())
    before = _lib.launch_count
    (grad,) = torch.autograd.grad(out, w, dy)
    assert (_lib.launch_count > before or tokens.numel() == 0) and grad.shape == w.shape and grad.dtype == w.dtype
    want, size, count = _sums(tokens, dy, V, scale, padding)
    # every addition is off by 2^-24 of the sizes at most, and so is the product with the scale
    tol = HALF_STEP[w.dtype] * want.abs() + SMALLEST[w.dtype] + (1 + HALF_STEP[w.dtype]) * size * 2.0 ** -24 * (count + 1)
    off = (grad.double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())
    assert grad[(count == 0)[:, 0]].eq(0).all()
    return grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,H,kind", [
    (1, 1, 1, "any"), (1, 5, 7, "any"), (0, 9, 16, "any"), (2, 3, 2, "same"), (31, 40, 33, "any"), (33, 2, 64, "any"), (64, 64, 8, "order"),
    (65, 64, 8, "same"), (200, 1000, 1001, "text"), (777, 50, 24, "runs"), (2048, 2048, 128, "order"), (3000, 70000, 50, "text"),
    (5000, 3, 40, "any"), (8193, 32000, 96, "text"), (20000, 300, 72, "same"), (20011, 140000, 16, "any"), (100003, 1000, 12, "text"),
    (300, 20, 9000, "any"), (70, 2 ** 20 + 3, 4, "any"), (40000, 513, 520, "text"), (256, 40, 24, "text"), (257, 40, 24, "text"),
    (256, 2 ** 18, 5, "same"), (1024, 600, 8, "runs"), (1025, 600, 8, "runs"), (32768, 2000, 8, "text"), (32769, 2000, 8, "text"), (5000, 511, 20, "runs"),
    (4096, 512, 16, "same")])
def test_table(n, V, H, kind, dtype):
    """One token to many (256, 1024 and 32,768 are the most that are not sorted, sorted by one block, and kept on the chip), tables of one
    row to a million, rows of one value to nine thousand, segments of every length."""
    g = torch.Generator(device=DEV).manual_seed(n + V)
    tokens = _tokens(n, V, kind, g)
    weight = torch.randn(V, H, generator=g, device=DEV).to(dtype)
    dy = torch.randn(n, H, generator=g, device=DEV).to(dtype)
    a = _check(tokens, weight, dy)
    b = _check(tokens.int(), weight, dy, scale=1.0)
    assert torch.equal(a, b)
    _check(tokens, weight, dy, scale=-7.3, padding=V // 2)


def test_all_tokens_are_padding():
    g = torch.Generator(device=DEV).manual_seed(0)
    weight, dy = torch.randn(11, 40, generator=g, device=DEV), torch.randn(300, 40, generator=g, device=DEV)
    assert _check(torch.full((300,), 4, device=DEV), weight, dy, 2.0, 4).eq(0).all()
    w = weight.requires_grad_()
    out = ops.embedding(torch.full((300,), 4, device=DEV), w, padding_idx=-7)
    assert torch.autograd.grad(out, w, dy)[0].eq(0).all()
    tokens = torch.randint(0, 2, (300,), generator=g, device=DEV) * 4
    _check(tokens, weight, dy, 2.0, 4)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    """Tokens of any shape and layout; tables with gaps between rows, off 16 bytes, turned; gradients of rows likewise and stretched."""
    g = torch.Generator(device=DEV).manual_seed(0)
    tokens = torch.randint(0, 60, (5, 7), generator=g, device=DEV)
    weight = torch.randn(60, 100, generator=g, device=DEV).to(dtype)
    dy = torch.randn(5, 7, 100, generator=g, device=DEV).to(dtype)
    flat = torch.empty(60 * 100 + 1, dtype=dtype, device=DEV)
    flat[1:] = weight.reshape(-1)
    _check(tokens, weight[:, :64], dy[..., :64])
    _check(tokens, weight[:, 3:72], dy[..., 5:74])
    _check(tokens, weight[::2], dy, padding=0) if int(tokens.max()) < 30 else _check(tokens % 30, weight[::2], dy, padding=0)
    _check(tokens, flat[1:].view(60, 100), dy, 3.0)
    _check(tokens, weight.t().contiguous().t(), dy.transpose(0, 2).contiguous().transpose(0, 2))
    _check(tokens.t(), weight, dy.transpose(0, 1))
    _check(tokens[:, ::2], weight, dy[:, ::2])
    _check(tokens[2, 3], weight, dy[2, 3])
    _check(tokens, weight, dy[0, 0].expand(5, 7, 100))
    w = weight.clone().requires_grad_()
    (grad,) = torch.autograd.grad(ops.embedding(tokens, w).sum(), w)
    assert torch.equal(grad[:, 0].float(), torch.bincount(tokens.reshape(-1), minlength=60).float())


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_tokens_outside_the_table(index):
    weight = torch.randn(10, 24, device=DEV, requires_grad=True)
    tokens = torch.tensor([3, -1, 10, 9, 2 ** 31 - 1, -2 ** 31, 3], device=DEV).to(index)
    if index == torch.int64:
        tokens = torch.cat([tokens, torch.tensor([1 << 40, -(1 << 40), (1 << 32) + 3], device=DEV)])
    out = ops.embedding(tokens, weight)
    inside = (tokens >= 0) & (tokens < 10)
    assert torch.equal(out.isnan().all(-1), ~inside) and torch.equal(out[inside], weight[tokens[inside].long()])
    dy = torch.randn_like(out)
    (grad,) = torch.autograd.grad(out, weight, dy)
    assert (grad.double() - _sums(tokens, dy, 10, 1.0)[0]).abs().max() < 1e-6 and grad[[0, 1, 2, 4, 5, 6, 7, 8]].eq(0).all()


def test_same_bits_every_time_and_on_another_stream():
    g = torch.Generator(device=DEV).manual_seed(0)
    tokens = _tokens(30000, 5000, "text", g)
    weight, dy = torch.randn(5000, 264, generator=g, device=DEV, requires_grad=True), torch.randn(30000, 264, generator=g, device=DEV)
    grad = lambda: torch.autograd.grad(ops.embedding(tokens, weight, 1.5, 3), weight, dy)[0]  # noqa: E731
    want = grad()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = grad()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and torch.equal(grad(), want)


def test_captured_into_graphs():
    """Two graphs, forward and backward, replayed in turn on new tokens."""
    g = torch.Generator(device=DEV).manual_seed(0)
    weight = torch.randn(900, 136, generator=g, device=DEV).bfloat16().requires_grad_()
    tokens, dy = torch.zeros(4, 700, dtype=torch.int64, device=DEV), torch.randn(4, 700, 136, generator=g, device=DEV).bfloat16()

    def both():
        out = ops.embedding(tokens, weight, 2.0, 1)
        return [out, *torch.autograd.grad(out, weight, dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(both())
    for kind in ("text", "any", "same"):
        tokens.copy_(_tokens(2800, 900, kind, g).view(4, 700))
        want = both()
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_gradients_of_gradients():
    """Lookups of the table that the gradient is asked with, and differences of the whole."""
    g = torch.Generator(device=DEV).manual_seed(0)
    tokens = torch.tensor([[1, 4, 1], [2, 0, 4]], device=DEV)
    w = torch.randn(6, 5, generator=g, device=DEV, requires_grad=True)
    out = ops.embedding(tokens, w, 1.5, 2)
    (gw,) = torch.autograd.grad(out.pow(3).sum(), w, create_graph=True)
    u = torch.randn_like(w)
    (ggw,) = torch.autograd.grad((gw * u).sum(), w)
    w64 = w.detach().double().requires_grad_()
    ref = torch.nn.functional.embedding(tokens, w64, 2) * 1.5
    (gr,) = torch.autograd.grad(ref.pow(3).sum(), w64, create_graph=True)
    (ggr,) = torch.autograd.grad((gr * u.double()).sum(), w64)
    assert (gw - gr).abs().max() < 1e-4 and (ggw - ggr).abs().max() < 1e-4


def test_tables_beyond_2_31_values():
    V, H = 131072, 16400
    weight = torch.zeros(V, H, dtype=torch.bfloat16, device=DEV)
    weight[-2:] = torch.randn(2, H, device=DEV).bfloat16()
    weight.requires_grad_()
    tokens = torch.tensor([V - 1, 0, V - 2, V - 1], device=DEV)
    out = ops.embedding(tokens, weight)
    assert torch.equal(out, weight.detach()[tokens])
    dy = torch.randn_like(out)
    (grad,) = torch.autograd.grad(out, weight, dy)
    assert torch.equal(grad[V - 2], dy[2]) and torch.equal(grad[0], dy[1]) and torch.equal(grad[V - 1], (dy[0].float() + dy[3].float()).bfloat16())
    assert grad[1:V - 2].eq(0).all()


def test_refusals():
    w, t = torch.randn(4, 8, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    for bad in (lambda: ops.embedding(t.cpu(), w), lambda: ops.embedding(t.float(), w), lambda: ops.embedding(t, w.double()), lambda: ops.embedding(t, w[0]),
                lambda: ops.embedding(t, w, float("nan")), lambda: ops.embedding(t, w, padding_idx=4), lambda: ops.embedding(t, w, padding_idx=-5)):
        with pytest.raises(ValueError):
            bad()
