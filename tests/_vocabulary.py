"""Plain 64-bit forms of the vocabulary's operators, and how far 32-bit kernels may be from them."""

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALLEST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}      # half a step there (32 bits: flushed)


def told(logits, tokens=None, top=0, temperature=1.0, ignore_index=-100):
    """{name: 64-bit tensor} of ``token_log_probs``, on the CPU."""
    z = logits.detach().cpu()
    y = z.double()
    y = (y - y.amax(-1, keepdim=True)) / temperature      # first: 64 bits do not hold log 2 beside 1e38
    log_p = y - torch.logsumexp(y, -1, keepdim=True)
    broken = (z.isnan() | (z == math.inf)).any(-1) | (z == -math.inf).all(-1)
    log_p[broken] = math.nan
    p = log_p.exp()
    keep = torch.ones(z.shape[:-1], dtype=torch.bool) if tokens is None else tokens.cpu() != ignore_index
    out = dict(log_p=log_p, p=p, keep=keep)
    entropy = -torch.where(p == 0, 0.0, p * log_p).sum(-1)
    out["entropy"] = torch.where(keep, entropy, 0.0)
    if tokens is not None:
        t, V = tokens.cpu(), z.shape[-1]
        inside = (t >= 0) & (t < V)
        lp = torch.where(inside, log_p.gather(-1, t.clamp(0, V - 1)[..., None])[..., 0], math.nan)
        out["log_probs"] = torch.where(keep, lp, 0.0)
    if top:
        at = torch.where(z.isnan(), math.nan, z).float().sort(dim=-1, descending=True, stable=True).indices[..., :top]
        out["top_tokens"] = torch.where(keep[..., None], at, -1)
        out["top_log_probs"] = torch.where(keep[..., None], log_p.gather(-1, at), 0.0)
    return out


def told_gradient(logits, tokens=None, d_log_probs=None, d_entropy=None, d_top=None, temperature=1.0, ignore_index=-100):
    """(gradient of the logits, sum of the sizes of what it is the sum of), 64-bit, on the CPU."""
    V = logits.shape[-1]
    w = told(logits, tokens, 0 if d_top is None else d_top.shape[-1], temperature, ignore_index)
    c, size = torch.zeros_like(w["p"]), torch.zeros_like(w["p"])
    given = []
    if d_log_probs is not None:
        t = tokens.cpu()
        g = torch.where((t >= 0) & (t < V) | ~w["keep"], d_log_probs.cpu().double(), math.nan)
        given.append((t.clamp(0, V - 1)[..., None], g[..., None]))
    if d_top is not None:
        given.append((w["top_tokens"].clamp(min=0), d_top.cpu().double()))
    for at, g in given:
        c.scatter_add_(-1, at, g)
        size.scatter_add_(-1, at, g.abs())
        size += w["p"] * g.abs().sum(-1, keepdim=True)
    c = c - w["p"] * c.sum(-1, keepdim=True)
    if d_entropy is not None:
        h, H = d_entropy.cpu().double()[..., None], w["entropy"][..., None]
        c -= torch.where(w["p"] == 0, w["p"] * 0, h * w["p"] * (w["log_p"] + H))
        size += torch.where(w["p"] == 0, w["p"] * 0, h.abs() * w["p"] * (w["log_p"].abs() + H))
    keep = w["keep"][..., None]
    return torch.where(keep, c / temperature, 0.0), torch.where(keep, size / temperature, 0.0)


def sum_error(V):
    """Relative error of a 32-bit sum of exponentials over a vocabulary, at worst: V / 256 additions one after another and some twenty of
    partial sums, each off by 2^-24 of the sum; the terms by 2^-22 (the exponential) and, on average, by the rounding of an exponent
    of log2 V or so."""
    return 2.0 ** -24 * (V / 256 + 20 + 4 + math.log2(max(V, 2)))


def check_told(got, want, V, top=0):
    """Statistics within the error of their sums; numbers of tokens and NaN exactly."""
    e = sum_error(V)
    for name in ("log_probs", "entropy", "top_log_probs"):
        g = getattr(got, name)
        if g is None:
            continue
        assert g.dtype == torch.float32 and g.shape == want[name].shape
        g, w = g.detach().cpu().double(), want[name].float().double()       # what 32 bits do not hold is infinite
        assert torch.equal(g.isnan(), w.isnan()), name
        fine = w.isfinite()
        assert torch.equal(g[~fine & ~w.isnan()], w[~fine & ~w.isnan()]), name
        # the logarithm of the sum takes its relative error; a difference of logits and the result are rounded, 2^-24 each; the mean that
        # the entropy has beside it is off by as much of itself as both of its sums are
        tol = e + 3 * 2.0 ** -24 * w[fine].abs() + (2 * e * (w[fine].abs() + 1) if name == "entropy" else 0)
        off = (g - w)[fine].abs()
        assert bool((off <= tol).all()), (name, float((off - tol).max()), float(off.max()))
    if top:
        assert got.top_tokens.dtype == torch.int64 and torch.equal(got.top_tokens.cpu(), want["top_tokens"])


def check_gradient(got, want, size, V, log_p):
    """Terms are off by the error of the probabilities (the sum, the exponential, the rounding of its exponent), the sum by a few
    roundings of 32 bits, the result by one of its own type.  A probability below 2^-126 is flushed to zero: off by that times the sizes
    of the gradients, at most 33 of a token and one of an entropy times an exponent of 126 or so, all of them below 5: 2^-116."""
    g = got.detach().cpu().double()
    assert torch.equal(g.isnan(), want.isnan())
    fine = want.isfinite()
    exponent = log_p.nan_to_num(0.0, neginf=0.0).abs()[fine]               # rows that are left out may have none
    tol = HALF_STEP[got.dtype] * want[fine].abs() + SMALLEST[got.dtype] + 2.0 ** -116 + size[fine] * (3 * sum_error(V) + 2.0 ** -24 * (16 + 4 * exponent))
    tol = tol * (1 + HALF_STEP[got.dtype])
    off = (g[fine] - want[fine]).abs()
    assert bool((off <= tol).all()), (float((off - tol).max()), float(off.max()))
