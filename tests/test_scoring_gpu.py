"""The vocabulary's two operators in the package's models: layers that look rows up, scored sequences, a policy-gradient step; the native
host paths against the Python code beside them; a slice of a vocabulary."""

import pytest
import torch
import torch.distributed as dist
import torch.nn.functional as F

from axonn_b200 import ops
from axonn_b200.ops import _lib

from _vocabulary import check_gradient, check_told, told, told_gradient

pytestmark = pytest.mark.gpu
DEV = "cuda"


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
    with torch.no_grad():
        model.head.proj.weight.mul_(10)
    return model.to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("expert_mode", [True, False])
def test_embedding_layer(dtype, expert_mode):
    from axonn_b200.intra_layer import Embedding

    torch.manual_seed(0)
    layer = Embedding(300, 72, padding_idx=5, expert_mode=expert_mode, dtype=dtype, scale=2.5).to(DEV)
    tokens = torch.randint(0, 300, (4, 33), device=DEV)
    tokens[:, ::5] = 5
    before = _lib.launch_count
    out = layer(tokens)
    assert _lib.launch_count > before
    w = layer.weight.detach().view(300, 72)
    assert torch.equal(out, (w[tokens].float() * 2.5).to(dtype))
    dy = torch.randn_like(out)
    out.backward(dy)
    keep = (tokens != 5).reshape(-1)
    want = torch.zeros(300, 72, dtype=torch.float64, device=DEV).index_add_(0, tokens.reshape(-1)[keep], dy.reshape(-1, 72)[keep].double(), alpha=2.5)
    # as many terms as a token occurs, rounded to the type once
    assert ((layer.weight.grad.view(300, 72).double() - want).abs() <= 2.0 ** (-8 if dtype == torch.bfloat16 else -20) * want.abs() + 1e-5).all()
    with torch.no_grad():
        assert torch.equal(layer(tokens.int()), out)
        assert torch.equal(layer.rows(3, 7, DEV), (w[3:10].float() * 2.5).to(dtype))


def test_embedding_layers_that_the_kernels_do_not_serve():
    from axonn_b200.intra_layer import Embedding

    torch.manual_seed(0)
    tokens = torch.randint(0, 50, (70,), device=DEV)
    for kw in (dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(dtype=torch.float64)):
        layer = Embedding(50, 16, expert_mode=True, **kw).to(DEV)
        before = _lib.launch_count
        with torch.set_grad_enabled("max_norm" not in kw):
            out = layer(tokens)
            assert _lib.launch_count == before
            if "max_norm" not in kw:
                out.sum().backward()
        kw.pop("dtype", None)
        w = layer.weight.detach().view(50, 16).clone().requires_grad_()
        ref = F.embedding(tokens, w if "max_norm" not in kw else w.detach(), **kw)
        assert torch.equal(out, ref)
        if "max_norm" not in kw:
            ref.sum().backward()
            assert torch.equal(layer.weight.grad.view(50, 16), w.grad)


@pytest.mark.parametrize("family", ["gpt", "llama"])
def test_scored_sequences(family):
    from axonn_b200.models import score_tokens

    model, g = _model(family).eval(), torch.Generator(device=DEV).manual_seed(1)
    tokens = torch.randint(0, 1000, (5, 77), generator=g, device=DEV)
    lengths = torch.tensor([77, 1, 40, 2, 76], device=DEV)
    with torch.no_grad():
        got = score_tokens(model, tokens, lengths, entropy=True, top=5, temperature=1.3)
        logits = model(tokens)[:, :-1]
    targets = tokens[:, 1:].masked_fill(torch.arange(1, 77, device=DEV) >= lengths[:, None], -100)
    check_told(got, told(logits, targets, 5, 1.3), 1000, 5)
    assert got.log_probs[1].eq(0).all() and got.top_tokens[1].eq(-1).all() and bool((got.log_probs[0] < 0).all())


@pytest.mark.parametrize("family", ["gpt", "llama"])
def test_policy_gradient_step(family):
    """Lookup, blocks, head, log-probabilities and entropy, and back into the table: the loss and the gradients beside those with a
    32-bit softmax in their place.  Both round the logits' gradients to bf16 once (2^-9 of a value on either side); behind that two
    layers of some eight operations round what has changed, 2^-8 each."""
    from axonn_b200.models import score_tokens

    model, g = _model(family), torch.Generator(device=DEV).manual_seed(1)
    tokens = torch.randint(0, 1000, (4, 65), generator=g, device=DEV)
    lengths = torch.tensor([65, 3, 50, 64], device=DEV)
    advantage = torch.randn(4, 64, generator=g, device=DEV)
    keep = torch.arange(1, 65, device=DEV) < lengths[:, None]
    r = score_tokens(model, tokens, lengths, entropy=True, top=2)
    loss = -(advantage * r.log_probs).sum() - 0.1 * r.entropy.sum() - 0.05 * r.top_log_probs.sum()
    loss.backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    logits = model(tokens)[:, :-1].float()
    log_p = logits.log_softmax(-1)
    entropy = -(log_p.exp() * log_p).sum(-1)
    best = log_p.gather(-1, r.top_tokens.clamp(min=0))
    plain = (-(advantage * log_p.gather(-1, tokens[:, 1:, None])[..., 0]) * keep - 0.1 * entropy * keep).sum() - 0.05 * (best * keep[..., None]).sum()
    assert abs(float(loss - plain)) <= 1e-4 * abs(float(plain)) + 1e-3
    plain.backward()
    for n, p in model.named_parameters():
        assert (got[n] - p.grad).float().norm() <= 16 * 2.0 ** -8 * p.grad.float().norm() + 1e-6, n
    unseen = torch.ones(1000, dtype=torch.bool, device=DEV)
    unseen[tokens.reshape(-1)] = False
    assert got["tok_emb.weight"].view(1000, -1)[unseen].eq(0).all()


def _python(monkeypatch, fn):
    with monkeypatch.context() as m:
        m.setattr(_lib, "_HOST", None)
        return fn()


@pytest.mark.parametrize("shape,form", [((9,), 0), ((5, 40), 0), ((3, 7, 33), 0), ((3, 7, 33), 1), ((2, 2, 3, 16), 0), ((0, 8), 0), ((4, 600), 2)])
def test_native_host_paths(shape, form, monkeypatch):
    """The same bits from C++ and from Python, with and without gradients, for all that either takes."""
    assert _lib.host() is not None
    torch.manual_seed(2)
    z0 = torch.randn(shape, device=DEV).bfloat16()
    if form == 1:
        z0 = z0[:, 1:]
    if form == 2:
        z0 = z0.t().contiguous().t()
    tokens = torch.randint(-1, z0.shape[-1] + 1, z0.shape[:-1], device=DEV)
    d = [torch.randn(z0.shape[:-1], device=DEV), torch.randn(z0.shape[:-1], device=DEV), torch.randn(*z0.shape[:-1], 3, device=DEV)]

    def probs(grad, given, which):
        z = z0.detach().requires_grad_(grad)
        r = ops.token_log_probs(z, tokens if given else None, entropy=True, top=3, temperature=0.8)
        out = [t for t in r if t is not None]
        if grad:
            outs = [(t, g) for i, (t, g) in enumerate(zip(r, d)) if t is not None and i in which]
            out += torch.autograd.grad([t for t, _ in outs], z, [g for _, g in outs])
        return out

    for grad, given, which in ((False, True, ()), (False, False, ()), (True, True, (0, 1, 2)), (True, False, (1, 2)), (True, True, (2,))):
        for a, b in zip(probs(grad, given, which), _python(monkeypatch, lambda: probs(grad, given, which))):
            assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.equal(a.isnan(), b.isnan())

    table = torch.randn(11, 24, device=DEV)
    ids = torch.randint(0, 11, shape[:-1], device=DEV)

    def rows(grad, scale, padding):
        w = table.detach().requires_grad_(grad)
        out = ops.embedding(ids, w, scale, padding)
        return [out] + (list(torch.autograd.grad(out, w, torch.ones_like(out) * 0.37)) if grad else [])

    for grad, scale, padding in ((False, 1.0, None), (True, 1.5, 3), (True, 1.0, -1), (False, 2.0, -1)):
        a, b = rows(grad, scale, padding), _python(monkeypatch, lambda: rows(grad, scale, padding))
        assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_seen_by_hooks_and_refused(monkeypatch):
    """Saved tensors in another layout, second backward passes, function transforms, inference mode."""
    z = torch.randn(6, 50, device=DEV, requires_grad=True)
    t = torch.randint(0, 50, (6,), device=DEV)
    w, ids = torch.randn(9, 8, device=DEV, requires_grad=True), torch.randint(0, 9, (30,), device=DEV)
    d, dy = torch.randn(6, device=DEV), torch.randn(30, 8, device=DEV)
    for python in (False, True):
        with monkeypatch.context() as m:
            if python:
                m.setattr(_lib, "_HOST", None)
            (gz,), (gw,) = torch.autograd.grad(ops.token_log_probs(z, t).log_probs, z, d), torch.autograd.grad(ops.embedding(ids, w), w, dy)
            turned = lambda x: x.t().contiguous().t() if x.dim() == 2 else x  # noqa: E731
            with torch.autograd.graph.saved_tensors_hooks(lambda x: turned(x.detach()), lambda x: x):
                r, e = ops.token_log_probs(z, t).log_probs, ops.embedding(ids, w)
            assert torch.equal(torch.autograd.grad(r, z, d)[0], gz) and torch.equal(torch.autograd.grad(e, w, dy)[0], gw)
            r, e = ops.token_log_probs(z, t).log_probs, ops.embedding(ids, w)
            for k in range(2):                             # a graph that is kept gives the same again
                assert torch.equal(torch.autograd.grad(r, z, d, retain_graph=k == 0)[0], gz)
                assert torch.equal(torch.autograd.grad(e, w, dy, retain_graph=k == 0)[0], gw)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(r, z, d)
            e = ops.embedding(ids, w)
            ids.add_(0)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(e, w, dy)
            with pytest.raises(RuntimeError):
                torch.func.grad(lambda x: ops.token_log_probs(x, t).log_probs.sum())(z.detach())
            assert torch.allclose(torch.func.grad(lambda x: (ops.embedding(ids, x) * dy).sum())(w.detach()), gw, atol=1e-5)
            with torch.inference_mode():
                assert torch.equal(ops.token_log_probs(z, t).log_probs, ops.token_log_probs(z.detach(), t).log_probs)
                assert torch.equal(ops.embedding(ids, w), w.detach()[ids])


@pytest.mark.parametrize("parts", [2, 5])
@pytest.mark.parametrize("rows,V", [(3, 4001), (300, 130), (2, 50)])
def test_a_slice_of_a_vocabulary(rows, V, parts):
    """Statistics and best logits of every slice, put together as the ranks do it, and the gradient of every slice."""
    from axonn_b200.ops import token_probs

    g = torch.Generator(device=DEV).manual_seed(V)
    whole = torch.randn(rows, V * parts, generator=g, device=DEV).bfloat16()
    whole[0, :V] = float("-inf")
    whole[-1, 3] = whole[-1, V + 1]                        # equal ones in two slices
    tokens = torch.randint(0, V * parts, (rows,), generator=g, device=DEV)
    tokens[1] = -100
    K, L, scale = 6, _lib.lib(), 1 / 0.9
    slices, stats, best, at = [whole[:, i * V:(i + 1) * V].contiguous() for i in range(parts)], [], [], []
    for i, z in enumerate(slices):
        s, b, a = torch.empty(rows, 4, device=DEV), torch.empty(rows, K, device=DEV), torch.empty(rows, K, dtype=torch.int64, device=DEV)
        _lib.check(L.axb_token_log_probs(z.data_ptr(), 0, V, tokens.data_ptr(), 0, 1, None, None, b.data_ptr(), a.data_ptr(), s.data_ptr(), 1, rows, V,
                                         i * V, V * parts, K, scale, -100, 0, 0, _lib.stream()), "axb_token_log_probs")
        stats.append(s.double()), best.append(b), at.append(a)
    m = torch.stack([s[:, 0] for s in stats]).amax(0)
    f = [((s[:, 0] - m) * scale).exp() for s in stats]
    total = sum(s[:, 1] * x for s, x in zip(stats, f))
    w = sum(torch.where(x > 0, x * (s[:, 2] + s[:, 1] * (s[:, 0] - m) * scale), 0) for s, x in zip(stats, f))
    zt = sum(s[:, 3] for s in stats)
    top, numbers = token_probs._best(torch.cat(best, 1), torch.cat(at, 1), K)
    joined = torch.stack([m, total, w, zt], -1)
    log_probs, H, top_log_probs, top_tokens, kept = token_probs._finish(joined, top.double(), numbers, tokens, True, K, scale, -100, (rows,))
    want = told(whole, tokens, K, 0.9)
    check_told(ops.TokenLogProbs(log_probs, H, top_log_probs, top_tokens), want, V * parts, K)
    d = [torch.randn(rows, generator=g, device=DEV), torch.randn(rows, generator=g, device=DEV), torch.randn(rows, K, generator=g, device=DEV)]
    full, size = told_gradient(whole, tokens, *d, temperature=0.9)
    for i, z in enumerate(slices):
        out = torch.empty_like(z)
        _lib.check(L.axb_token_log_probs_bwd(z.data_ptr(), 0, V, tokens.data_ptr(), 0, 1, kept.data_ptr(), *(x.data_ptr() for x in d), top_tokens.data_ptr(),
                                             out.data_ptr(), 1, rows, V, i * V, V * parts, K, scale, -100, 0, _lib.stream()), "axb_token_log_probs_bwd")
        cut = slice(i * V, (i + 1) * V)
        check_gradient(out, full[:, cut], size[:, cut], V * parts, want["log_p"][:, cut])
