"""Calls of the vocabulary's operators, and of the functions on them, at the ends of what they take: on a GPU."""

import pytest
import torch
import torch.distributed as dist

from axonn_b200 import ops
from axonn_b200.ops import _lib

from _vocabulary import HALF_STEP, SMALLEST, check_told, told
from _vocabulary_ends import COLD, HOT, check_ends_of_temperature, ends_of_temperature

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module", autouse=True)
def _grid():
    from axonn_b200 import axonn as ax

    if not dist.is_initialized():
        dist.init_process_group("nccl", store=dist.HashStore(), rank=0, world_size=1)
    if not ax.is_initialized:
        ax.init(G_inter=1, G_data=1, G_intra_r=1, G_intra_c=1, G_intra_d=1)


def _model(family):
    from axonn_b200.models import GPT, GPTConfig, Llama, LlamaConfig

    torch.manual_seed(0)
    shape = dict(n_layers=2, hidden=256, n_heads=4, ffn=512, vocab=1000, seq_len=256)
    model = GPT(GPTConfig(**shape), dtype=torch.bfloat16) if family == "gpt" else Llama(LlamaConfig(n_kv_heads=2, **shape), dtype=torch.bfloat16)
    return model.to(DEV)


@pytest.mark.parametrize("family", ["gpt", "llama"])
def test_padding_outside_the_table(family):
    """What stands behind the rows' ends is no token: any number may, and neither the results nor the gradients see it."""
    from axonn_b200.models import beam_generate, greedy_generate, score_tokens

    model, g = _model(family), torch.Generator(device=DEV).manual_seed(1)
    tokens, lengths = torch.randint(0, 1000, (4, 77), generator=g, device=DEV), torch.tensor([77, 40, 2, 1], device=DEV)
    behind = torch.arange(77, device=DEV) >= lengths[:, None]

    def scored(t):
        model.zero_grad(set_to_none=True)
        r = score_tokens(model, t, lengths, entropy=True, top=3)
        (r.log_probs.sum() + r.entropy.sum()).backward()
        return [x.detach() for x in r] + [p.grad for p in model.parameters()]

    def generated(t):
        return [greedy_generate(model, t, 5, cache_dtype=torch.int8, prompt_lengths=lengths),
                *beam_generate(model, t, 5, 3, cache_dtype=torch.int8, prompt_lengths=lengths)]

    for call in (scored, generated):
        want = call(tokens.masked_fill(behind, 0))
        assert all(bool(x.isfinite().all()) for x in want)
        for pad in (-1, -100, 1000, 1 << 40):
            assert all(torch.equal(a, b) for a, b in zip(call(tokens.masked_fill(behind, pad)), want)), pad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [COLD, HOT])
def test_ends_of_the_temperature(dtype, temperature, monkeypatch):
    check_ends_of_temperature(*ends_of_temperature(dtype, DEV), temperature)
    monkeypatch.setattr(_lib, "_HOST", None)
    check_ends_of_temperature(*ends_of_temperature(dtype, DEV), temperature)


def test_temperatures_that_are_refused():
    logits, tokens = ends_of_temperature(torch.float32, DEV)
    for temperature in (1e-39, 3e-39, COLD / 2, 2 * HOT, 9e37, 3e38, 0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_log_probs(logits, tokens, temperature=temperature)


def test_gradient_of_wide_tables():
    """More blocks of columns than a grid has rows of blocks.  Small whole numbers, whose sums are exact."""
    V, H, n = 3, 65535 * 128 + 8, 300
    g = torch.Generator(device=DEV).manual_seed(0)
    weight = torch.randn(V, H, generator=g, device=DEV).bfloat16().requires_grad_()
    tokens = torch.cat([torch.ones(200, dtype=torch.int64, device=DEV), torch.randint(0, V, (n - 200,), generator=g, device=DEV)])
    dy = torch.randint(-3, 4, (H,), generator=g, device=DEV).bfloat16().expand(n, H)
    out = ops.embedding(tokens, weight)
    assert torch.equal(out[::37], weight.detach()[tokens[::37]])
    (grad,) = torch.autograd.grad(out, weight, dy)
    for v, count in enumerate(torch.bincount(tokens, minlength=V).tolist()):
        assert torch.equal(grad[v], (dy[0].float() * count).bfloat16())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,H,kind", [(200, 40, "any"), (3000, 40, "any"), (3000, 33, "same"), (5000, 6, "any")])
def test_numbers_below_the_smallest_normal_one(n, H, kind, dtype):
    """They are kept, as torch.nn.functional.embedding does it: their sums in 32 bits are exact (16-bit types: multiples of 2^-133 or 2^-24), a
    factor that is a power of two rounds nothing but the result.  The wanted ones come from 64 bits on the CPU, rounded once."""
    V, smallest, by = 50, torch.finfo(dtype).smallest_normal, 0.125
    g = torch.Generator().manual_seed(n + H)
    weight = (torch.randn(V, H, generator=g).double() * smallest * 2).to(dtype)
    tokens = torch.full((n,), 7) if kind == "same" else torch.randint(0, V, (n,), generator=g)
    dy = (torch.randn(n, H, generator=g).double() * smallest / 64).to(dtype)
    assert bool((weight.abs() < smallest).any()) and bool((dy.abs() < smallest).any()) and dy.count_nonzero() > n * H / 4
    for scale in (1.0, by):
        w = weight.to(DEV).requires_grad_()
        out = ops.embedding(tokens.to(DEV), w, scale)
        assert torch.equal(out.cpu(), (weight.double() * scale).to(dtype)[tokens])
        (grad,) = torch.autograd.grad(out, w, dy.to(DEV))
        want, size = (torch.zeros(V, H, dtype=torch.float64).index_add_(0, tokens, d) * scale for d in (dy.double(), dy.double().abs()))
        # fp32 has 24 bits above 2^-149: sums up to 2^-125 are exact, larger ones of n terms off by n times 2^-24 of their terms' sizes
        tol = torch.where(size / scale > 2.0 ** -125, n * 2.0 ** -24 * size, 0.0) if dtype == torch.float32 else torch.zeros_like(want)
        assert bool(((grad.cpu().double() - want.to(dtype).double()).abs() <= tol).all())


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,kind", [(1, "any"), (150, "any"), (3000, "any"), (700, "same")])
def test_batched_gradients(n, kind, dtype, native, monkeypatch):
    """Many gradients of the rows at once, as of torch.nn.functional.embedding; tokens outside the table and padding have none."""
    if not native:
        monkeypatch.setattr(_lib, "_HOST", None)
    V, H, scale, pad = 40, 12, -1.5, 3
    g = torch.Generator(device=DEV).manual_seed(n)
    weight = torch.randn(V, H, generator=g, device=DEV).to(dtype).requires_grad_()
    tokens = torch.full((n,), 7, device=DEV) if kind == "same" else torch.randint(-2, V + 2, (n,), generator=g, device=DEV)
    dy = torch.randn(5, n, H, generator=g, device=DEV).to(dtype)
    for ids in (tokens, tokens.int()):
        out = ops.embedding(ids, weight, scale, pad)
        (got,) = torch.autograd.grad(out, weight, dy, is_grads_batched=True, retain_graph=True)
        assert got.shape == (5, V, H) and got.dtype == dtype
        there = (tokens >= 0) & (tokens < V) & (tokens != pad)
        for i in range(5):
            d, zero = dy[i][there].double(), torch.zeros(V, H, dtype=torch.float64, device=DEV)
            want, size = zero.index_add(0, tokens[there], d, alpha=scale), zero.index_add(0, tokens[there], d.abs(), alpha=abs(scale))
            count = torch.bincount(tokens[there], minlength=V)[:, None]
            # as of the single gradient: every addition and the product with the scale 2^-24 of the sizes, then the type's rounding
            tol = HALF_STEP[dtype] * want.abs() + SMALLEST[dtype] + (1 + HALF_STEP[dtype]) * size * 2.0 ** -24 * (count + 1)
            assert bool(((got[i].double() - want).abs() <= tol).all())


def test_vectorised_jacobians(monkeypatch):
    """The same with and without a loop over the rows, and gradients of batched gradients."""
    tokens = torch.tensor([[1, 4, 1], [2, 0, 4]], device=DEV)
    weight = torch.randn(6, 4, device=DEV)
    for native in (True, False):
        with monkeypatch.context() as m:
            if not native:
                m.setattr(_lib, "_HOST", None)
            f = lambda w: ops.embedding(tokens, w, 2.0, 2).square().sum(-1)  # noqa: E731
            a, b = (torch.autograd.functional.jacobian(f, weight, vectorize=v) for v in (True, False))
            assert torch.equal(a, b)
            w = weight.clone().requires_grad_()
            out = ops.embedding(tokens, w, 2.0, 2)
            u = torch.randn(3, 2, 3, 4, device=DEV, requires_grad=True)
            (g,) = torch.autograd.grad(out, w, u, is_grads_batched=True, create_graph=True)
            c = torch.randn_like(g)
            (gu,) = torch.autograd.grad(g, u, c)
            keep = (tokens != 2)[None, :, :, None]
            assert torch.equal(gu, 2.0 * c[:, tokens] * keep)


def test_batched_gradients_of_log_probabilities_are_refused(monkeypatch):
    z, t = torch.randn(6, 50, device=DEV, requires_grad=True), torch.randint(0, 50, (6,), device=DEV)
    for native in (True, False):
        with monkeypatch.context() as m:
            if not native:
                m.setattr(_lib, "_HOST", None)
            r = ops.token_log_probs(z, t, entropy=True)
            with pytest.raises(RuntimeError, match="batched gradients"):
                torch.autograd.grad(r.log_probs, z, torch.randn(3, 6, device=DEV), is_grads_batched=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,H", [(1, 1, 1), (1, 5, 7), (33, 2, 64), (200, 1000, 1001), (257, 40, 24), (3000, 700, 50), (20011, 1400, 16), (300, 20, 9000), (16384, 3000, 264)])
def test_lookups_are_copies(n, V, H, dtype):
    """Without a scale every bit is the table's, whatever the sizes and wherever the rows begin; with gradients and without."""
    g = torch.Generator(device=DEV).manual_seed(n + H)
    tokens = torch.randint(0, V, (n,), generator=g, device=DEV)
    flat = torch.randn(V * (H + 3) + 1, generator=g, device=DEV).to(dtype)
    dense, off, gaps = flat[:V * H].view(V, H), flat[1:1 + V * H].view(V, H), flat[1:].view(V, H + 3)[:, 2:2 + H]
    for table in (dense, off, gaps, dense.t().contiguous().t()):
        want = table[tokens]
        for ids in (tokens, tokens.int()):
            assert torch.equal(ops.embedding(ids, table), want)
            assert torch.equal(ops.embedding(ids, table.detach().requires_grad_()), want)


@pytest.mark.parametrize("rows", [1, 64, 300])
@pytest.mark.parametrize("V,dtype", [(1500, torch.bfloat16), (2048, torch.bfloat16), (2049, torch.float16), (4096, torch.float16), (4097, torch.bfloat16),
                                     (1024, torch.float32), (1025, torch.float32), (2048, torch.float32), (2049, torch.float32)])
def test_alternatives_of_few_narrow_rows(rows, V, dtype):
    """Rows that a warp takes and rows that a block takes, by their bytes and by how many alternatives are asked for."""
    g = torch.Generator(device=DEV).manual_seed(V + rows)
    logits = (3 * torch.randn(rows, V, generator=g, device=DEV)).to(dtype)
    logits[::3, V // 2:] = -float("inf")
    tokens = torch.randint(0, V // 2, (rows,), generator=g, device=DEV)
    for top in (1, 8, 9, 20, 21, 32):
        check_told(ops.token_log_probs(logits, tokens, entropy=True, top=top), told(logits, tokens, top), V, top)
