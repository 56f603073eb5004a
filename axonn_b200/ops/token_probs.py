"""Log-probabilities of given tokens, with the entropy and the best alternatives (``csrc/token_probs.cu``).

The logits are read once forward and once backward, in the type they have: neither their softmax nor a 32-bit copy of the
``[tokens, vocabulary]`` matrix is stored.  Statistics are 32-bit, added in an order that no timing changes: the same bits on every run."""

import math
from typing import NamedTuple, Optional

import torch
import torch.distributed as dist

from . import _lib
from .direct import batched, first_derivative_only, host_paths
from .gemm import as_written
from .kv_cache import _elsewhere

MOST_ALTERNATIVES = 32
_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
# Of temperatures; the hottest is its reciprocal.  32 bits hold the factor 1 / T, with log2 e and with gradients, as a normal number (one that is
# flushed to zero would make NaN of a masked token, one that overflows of the likeliest), and differences of logits that they do not
# hold (2^128) are no less than 2^28 beside a temperature: their exponential is zero.
_COLDEST = 2.0 ** -100


class TokenLogProbs(NamedTuple):
    """What ``token_log_probs`` says of every position: ``log_probs [...]``, ``entropy [...]`` and ``top_log_probs [..., top]`` (fp32)
    and ``top_tokens [..., top]`` (int64, best first); ``None`` for what was not asked for."""

    log_probs: Optional[torch.Tensor]
    entropy: Optional[torch.Tensor]
    top_log_probs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def token_log_probs(logits, tokens=None, entropy=False, top=0, temperature=1.0, group=None, ignore_index=-100):
    """Log-probabilities of ``tokens [...]`` (int64) under ``softmax(logits / temperature)``, ``logits [..., vocabulary]`` in bf16, fp16 or
    fp32: a ``TokenLogProbs``.  With ``entropy`` also that of each distribution, with ``top`` (up to 32) the log-probabilities and numbers
    of its likeliest tokens, equal ones in their order.  ``tokens=None``: the entropy and the alternatives alone.

    Positions whose token is ``ignore_index`` are not looked at: they give zeros, alternatives of -1, and no gradient.  Any other number
    outside the vocabulary gives NaN.  Logits of ``-inf`` are tokens that cannot come; a position that leaves none, or that has a NaN or
    ``+inf`` among its logits, is NaN throughout (a NaN counts as the largest logit among the alternatives).  On a GPU logits below
    2^-126 count as zero.  Temperatures go from 2^-100 to 2^100.

    Everything but ``top_tokens`` can be differentiated once, with one gradient at a time, by the logits, which may have any strides (such
    as ``logits[:, :-1]``) and are left as they are.  With ``group`` the last dimension is this rank's contiguous slice of the vocabulary, of
    equal size on all ranks (rank order = slice order); ``tokens`` and every result count the whole vocabulary, and the gradients of the
    results are those of all ranks, as for ``cross_entropy``.  Neither synchronises: calls without ``group`` can be captured into a CUDA
    graph."""
    if group is None and logits.is_cuda and temperature and (host := host_paths()) is not None:
        out = host.token_log_probs(logits, tokens, entropy, top, 1 / temperature, ignore_index)
        if out is not None:
            return TokenLogProbs(*out)
    dev = logits.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return token_log_probs(logits, tokens, entropy, top, temperature, group, ignore_index)
    if logits.dtype not in _DT or logits.ndim == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits must be [..., vocabulary] in bf16, fp16 or fp32, not {logits.dtype} {list(logits.shape)}")
    V = logits.shape[-1]
    if V > 1 << 30:
        raise ValueError(f"a vocabulary of at most {1 << 30}, not {V}")
    if not 0 <= top <= min(MOST_ALTERNATIVES, V):
        raise ValueError(f"0 to {min(MOST_ALTERNATIVES, V)} alternatives of {V} tokens, not {top}")
    if not _COLDEST <= temperature <= 1 / _COLDEST:
        raise ValueError(f"the temperature is a positive number from {_COLDEST:.1e} to {1 / _COLDEST:.1e}, not {temperature}")
    if tokens is None:
        if not entropy and not top:
            raise ValueError("without tokens there is something to say of the entropy or the alternatives only")
    else:
        if tokens.dtype != torch.int64 or tokens.shape != logits.shape[:-1]:
            raise ValueError(f"tokens must be int64 {list(logits.shape[:-1])}, not {tokens.dtype} {list(tokens.shape)}")
        if tokens.device != dev:
            raise ValueError(f"tensors on {dev} and {tokens.device}")
    out = _TokenLogProbsFn.apply(logits, tokens, bool(entropy), int(top), 1 / temperature, group, ignore_index)
    return TokenLogProbs(*out)


def _as_rows(t, dims):
    """``t`` as a view (a copy, where its strides allow none) with two dimensions in front of the last ``dims``, which are dense."""
    front = t.shape[:t.ndim - dims]
    if dims and t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    if len(front) > 2:
        rest = t.shape[t.ndim - dims:]
        try:
            t = t.view(-1, front[-1], *rest)
        except RuntimeError:
            t = t.reshape(-1, front[-1], *rest)
    while t.ndim < dims + 2:
        t = t[None]
    return t


def _forward_torch(logits, tokens, top, scale, start, total, ignored):
    """``stats [rows, 4]``, the alternatives' logits and numbers, of this slice of the vocabulary."""
    z = logits.detach().reshape(-1, logits.shape[-1])
    y = z.double()
    m = y.amax(-1)
    d = (y - m.masked_fill(m == -math.inf, 0)[:, None]) * scale
    e = d.exp()
    zt = torch.zeros_like(m)
    if tokens is not None:
        t = tokens.reshape(-1) - start
        inside = (t >= 0) & (t < z.shape[1])
        zt = torch.where(inside, y.gather(1, t.clamp(0, z.shape[1] - 1)[:, None])[:, 0], 0.0)
        zt = zt.masked_fill(((tokens.reshape(-1) < 0) | (tokens.reshape(-1) >= total)) & ~ignored, math.nan)
    stats = torch.stack([m, e.sum(-1), torch.where(e > 0, e * d, e).masked_fill(e == 0, 0).sum(-1), zt], -1)
    best, at = _best(z.float(), torch.arange(z.shape[1], device=z.device).expand_as(z), top)
    return stats, best.double(), at + start


def _best(z, numbers, top):
    """The ``top`` largest of ``z [rows, n]`` in the order of ``numbers``, a NaN as the largest."""
    at = torch.where(z.isnan(), math.nan, z).sort(dim=-1, descending=True, stable=True).indices[:, :top]
    return z.gather(1, at), numbers.gather(1, at)


def _of_all(stats, best, at, scale, top, group):
    """Statistics and alternatives of the whole vocabulary from those of the ranks' slices."""
    m, s, w, zt = stats.unbind(-1)
    most = m.masked_fill(m.isnan(), -math.inf)
    dist.all_reduce(most, op=dist.ReduceOp.MAX, group=group)
    shift = (m - most) * scale
    f = torch.where(m == -math.inf, 0, shift.exp())         # a slice without a token that can come adds nothing
    sums = torch.stack([s * f, torch.where(f > 0, f * (w + s * shift), 0), zt])
    dist.all_reduce(sums, group=group)
    if top:
        n = dist.get_world_size(group)
        values, numbers = (torch.empty((n,) + t.shape, dtype=t.dtype, device=t.device) for t in (best, at))
        dist.all_gather(list(values), best.contiguous(), group=group)
        dist.all_gather(list(numbers), at.contiguous(), group=group)
        best, at = _best(values.transpose(0, 1).flatten(1), numbers.transpose(0, 1).flatten(1), top)
    return torch.stack([most, *sums], -1), best, at


class _TokenLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, entropy, top, scale, group, ignore_index):
        n = 1 if group is None else dist.get_world_size(group)
        V, front, dev = logits.shape[-1], logits.shape[:-1], logits.device
        start = 0 if n == 1 else dist.get_rank(group) * V
        rows = logits.numel() // V
        ctx.scale, ctx.start, ctx.total, ctx.top, ctx.ignore_index = scale, start, n * V, top, ignore_index
        ctx.asked = (tokens is not None, entropy, top > 0)
        ctx.set_materialize_grads(False)
        if logits.is_cuda and rows > 0:
            z = _as_rows(logits.detach(), 1)
            t = None if tokens is None else _as_rows(tokens, 0)
            f32 = dict(dtype=torch.float32, device=dev)
            log_probs = torch.empty(front, **f32) if tokens is not None else None
            H = torch.empty(front, **f32) if entropy else None
            best = torch.empty(front + (top,), **f32) if top else None
            at = torch.empty(front + (top,), dtype=torch.int64, device=dev) if top else None
            stats = torch.empty(rows, 4, **f32)
            st = _lib.lib().axb_token_log_probs(
                z.data_ptr(), z.stride(0), z.stride(1), _lib.addr(t), *((0, 0) if t is None else t.stride()), _lib.addr(log_probs), _lib.addr(H),
                _lib.addr(best), _lib.addr(at), stats.data_ptr(), z.shape[0], z.shape[1], V, start, n * V, top, scale, ignore_index, n == 1,
                _DT[z.dtype], _lib.stream())
            _lib.check(st, "axb_token_log_probs")
            if n > 1:
                stats, best, at = _of_all(stats.double(), None if best is None else best.view(rows, top), None if at is None else at.view(rows, top),
                                            scale, top, group)
        else:
            ignored = torch.zeros(rows, dtype=torch.bool, device=dev) if tokens is None else tokens.reshape(-1) == ignore_index
            stats, best, at = _forward_torch(logits, tokens, top, scale, start, n * V, ignored)
            if n > 1:
                stats, best, at = _of_all(stats, best, at, scale, top, group)
        if not logits.is_cuda or rows == 0 or n > 1:
            log_probs, H, best, at, stats = _finish(stats, best, at, tokens, entropy, top, scale, ignore_index, front)
        ctx.save_for_backward(logits, tokens, stats, at)
        if at is not None:
            ctx.mark_non_differentiable(at)
        return log_probs, H, best, at

    @staticmethod
    @first_derivative_only
    def backward(ctx, d_log_probs, d_entropy, d_top, _):
        if any(map(batched, (d_log_probs, d_entropy, d_top))):
            raise RuntimeError("TokenLogProbs: batched gradients are not implemented")
        logits, tokens, stats, at = ctx.saved_tensors
        # what hooks (offloading, compression) give back may lie in another layout
        stats, at = as_written(stats), None if at is None else at.contiguous()
        if d_log_probs is None and d_entropy is None and d_top is None:
            return (None,) * 7
        V, rows = logits.shape[-1], logits.numel() // logits.shape[-1]
        d = [None if g is None else g.to(torch.float32).contiguous() for g in (d_log_probs, d_entropy, d_top)]
        if logits.is_cuda and rows > 0:
            z = _as_rows(logits.detach(), 1)
            t = None if tokens is None else _as_rows(tokens, 0)
            out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            st = _lib.lib().axb_token_log_probs_bwd(
                z.data_ptr(), z.stride(0), z.stride(1), _lib.addr(t), *((0, 0) if t is None else t.stride()), stats.data_ptr(), *map(_lib.addr, d),
                _lib.addr(at), out.data_ptr(), z.shape[0], z.shape[1], V, ctx.start, ctx.total, ctx.top, ctx.scale, ctx.ignore_index,
                _DT[z.dtype], _lib.stream())
            _lib.check(st, "axb_token_log_probs_bwd")
            return (out,) + (None,) * 6
        return (_backward_torch(ctx, logits, tokens, stats, at, *d),) + (None,) * 6


def _finish(stats, best, at, tokens, entropy, top, scale, ignore_index, front):
    """Results from the statistics of the whole vocabulary, and what the backward takes: (m, s, entropy, log s) of every row."""
    m, s, w, zt = stats.unbind(-1)
    H = s.log() - w / s
    ignored = None if tokens is None else tokens.reshape(-1) == ignore_index
    keep = (lambda t, other: t) if tokens is None else (lambda t, other: t.masked_fill(ignored.view([-1] + [1] * (t.ndim - 1)), other))
    log_probs = None if tokens is None else keep((zt - m) * scale - s.log(), 0).float().view(front)
    top_log_probs = keep((best - m[:, None]) * scale - s.log()[:, None], 0).float().view(*front, top) if top else None
    top_tokens = keep(at, -1).view(*front, top) if top else None
    return log_probs, keep(H, 0).float().view(front) if entropy else None, top_log_probs, top_tokens, torch.stack([m, s, H, s.log()], -1).float()


def _backward_torch(ctx, logits, tokens, stats, at, d_log_probs, d_entropy, d_top):
    V = logits.shape[-1]
    z = logits.reshape(-1, V)
    m, s, H = (t[:, None] for t in stats.double().unbind(-1)[:3])
    y = (z.double() - m) * ctx.scale
    p = y.exp() / s
    ignored = torch.zeros_like(m, dtype=torch.bool) if tokens is None else (tokens.reshape(-1) == ctx.ignore_index)[:, None]
    given = []                                         # (token within the slice, gradient of its log-probability)
    if d_log_probs is not None:
        t = tokens.reshape(-1, 1)
        outside = ((t < 0) | (t >= ctx.total)) & ~ignored
        given.append((t - ctx.start, d_log_probs.reshape(-1, 1).double().masked_fill(outside, math.nan)))
    if d_top is not None:
        given.append((at.reshape(-1, ctx.top) - ctx.start, d_top.reshape(-1, ctx.top).double()))
    out = torch.zeros_like(p)
    for token, g in given:
        out -= p * g.sum(-1, keepdim=True)
        inside = (token >= 0) & (token < V)
        out.scatter_add_(1, token.clamp(0, V - 1), torch.where(inside, g, 0))
    if d_entropy is not None:
        h = d_entropy.reshape(-1, 1).double()
        out -= torch.where(p > 0, p * h * (y - s.log() + H), p * 0)
    return (out * ctx.scale).masked_fill(ignored, 0).to(logits.dtype).view(logits.shape)
