"""The two ends of a language model's vocabulary: what is said of given tokens, and the table that tokens are looked up in.

``token_log_probs`` gives the log-probabilities of given tokens under ``[..., vocabulary]`` logits, with the entropy of the distribution
and its best alternatives where they are asked for; as a training step (policy gradients, distillation) with the gradient of the logits.
``embedding`` looks tokens up in a table and scales their rows; its gradient sums the rows of equal tokens.

Sizes are those of the package's own configurations (GPT-1.3B: hidden 2048, 2048 positions, vocabulary 50304; Llama-8B: hidden 4096, 4096
positions, vocabulary 128256; Mixtral: vocabulary 32000) and generic ones.
"""

import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORED = -100
LARGEST = 1e9                        # bytes of a drawn case's logits, or of its table


def listed():
    return [
        # the token that one request has got, with five alternatives: latency
        dict(name="decode_one_request", kind="score", rows=1, steps=1, vocab=32000, dtype="bf16", entropy=False, top=5, temperature=1.0,
             ignored=0.0, masked=0.0),
        # a decoding step of a full batch over Llama-8B's vocabulary, part of which a grammar rules out
        dict(name="decode_batch", kind="score", rows=64, steps=1, vocab=128256, dtype="bf16", entropy=True, top=20, temperature=0.8,
             ignored=0.0, masked=0.3),
        # prompts scored with GPT-1.3B: all positions but the last, ragged lengths
        dict(name="score_prompts", kind="score", rows=8, steps=2048, vocab=50304, dtype="bf16", entropy=False, top=0, temperature=1.0,
             ignored=0.15, masked=0.0),
        # 32-bit logits of an odd vocabulary, with alternatives
        dict(name="score_odd_vocabulary", kind="score", rows=1000, steps=1, vocab=49999, dtype="fp32", entropy=True, top=8, temperature=0.7,
             ignored=0.0, masked=0.0),
        # a short policy-gradient step: few rows
        dict(name="policy_few_rows", kind="policy", rows=3, steps=33, vocab=32000, dtype="fp16", entropy=True, top=0, temperature=1.0,
             ignored=0.2, masked=0.0),
        # a policy-gradient step with an entropy bonus over Llama-8B's vocabulary
        dict(name="policy_batch", kind="policy", rows=4096, steps=1, vocab=128256, dtype="bf16", entropy=True, top=0, temperature=1.0,
             ignored=0.1, masked=0.0),
        # the tokens of a decoding step, Llama-8B: latency
        dict(name="lookup_decode", kind="lookup", tokens=64, vocab=128256, hidden=4096, dtype="bf16", scale=1.0, padded=0.0, distinct=False),
        # a batch of prompts, GPT-1.3B, rows scaled by the root of their length
        dict(name="lookup_prompts", kind="lookup", tokens=16384, vocab=50304, hidden=2048, dtype="bf16", scale=45.25, padded=0.0,
             distinct=False),
        # learned positions of GPT-1.3B: every row once
        dict(name="table_positions", kind="table", tokens=2048, vocab=2048, hidden=2048, dtype="bf16", scale=1.0, padded=0.0, distinct=True),
        # a training batch of GPT-1.3B
        dict(name="table_batch", kind="table", tokens=16384, vocab=50304, hidden=2048, dtype="bf16", scale=1.0, padded=0.0, distinct=False),
        # a training batch of Llama-8B
        dict(name="table_large_vocabulary", kind="table", tokens=16384, vocab=128256, hidden=4096, dtype="bf16", scale=64.0, padded=0.0,
             distinct=False),
        # rows that are no whole number of 16 bytes, many equal padding tokens
        dict(name="table_padded_odd", kind="table", tokens=6001, vocab=32000, hidden=1001, dtype="fp32", scale=1.0, padded=0.4,
             distinct=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind, dtype = rng.choice(["score", "score", "policy", "lookup", "table", "table"]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("score", "policy"):
        vocab = _log(rng, 1000, 131072)
        top = rng.choice([0, 0, 1, rng.randint(2, 32)])
        count = _log(rng, 1, max(1, min(16384, int(LARGEST / (4 if top else 1) / (vocab * SIZE[dtype])))))
        steps = rng.choice([1, 1, _log(rng, 1, count)])
        return dict(kind=kind, rows=max(1, count // steps), steps=steps, vocab=vocab, dtype=dtype, entropy=rng.random() < 0.5,
                    top=top, temperature=rng.choice([1.0, rng.uniform(0.5, 1.5)]),
                    ignored=rng.choice([0.0, rng.uniform(0, 0.6)]), masked=rng.choice([0.0, 0.0, rng.uniform(0.1, 0.9)]))
    vocab, hidden = _log(rng, 500, 131072), rng.choice([_log(rng, 50, 8192), 64 * _log(rng, 1, 128)])
    vocab = min(vocab, int(LARGEST / (hidden * SIZE[dtype])))
    tokens = _log(rng, 1, max(1, min(65536, int(LARGEST / 8 / (hidden * SIZE[dtype])))))
    return dict(kind=kind, tokens=tokens, vocab=vocab, hidden=hidden, dtype=dtype, scale=rng.choice([1.0, math.sqrt(hidden)]),
                padded=rng.choice([0.0, 0.0, rng.uniform(0, 0.9)]), distinct=False)


# ----------------------------------------------------------------------------- inputs

def _kept(case):
    """Of every row, how many of its first positions count: a function of the case alone."""
    R, P, ignored = case["rows"], _positions(case), case["ignored"]
    if P == 1:
        return [int((i * 0.6180339887498949) % 1.0 >= ignored) for i in range(R)]
    return [max(0, P - int(2 * ignored * P * (i + 0.5) / R)) for i in range(R)]


def _positions(case):
    """Positions of a row that have a next token: all but the last, where there are several."""
    return case["steps"] - 1 if case["steps"] > 1 else 1


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, V, dtype = case["kind"], case["vocab"], TYPES[case["dtype"]]
    if kind in ("score", "policy"):
        R, S, P = case["rows"], case["steps"], _positions(case)
        logits = torch.empty(R, S, V, dtype=dtype, device=DEV).normal_(0, 2.5, generator=g)
        tokens = torch.randint(0, V, (R, S), generator=g, device=DEV)
        if case["masked"]:
            logits.masked_fill_(torch.rand(V, generator=g, device=DEV) < case["masked"], float("-inf"))
        # what is asked of is mostly likely
        at = tokens[:, -P:]
        likely = (8 * torch.rand(R, P, generator=g, device=DEV)).to(dtype)
        logits[:, :P].scatter_(2, at[..., None], likely[..., None])
        kept = torch.tensor(_kept(case), device=DEV)
        at[torch.arange(P, device=DEV) >= kept[:, None]] = IGNORED
        state = dict(case=case, logits=logits[:, :P], tokens=at)
        if kind == "policy":
            state["logits"].requires_grad_()
            state["d_log_probs"] = torch.randn(R, P, generator=g, device=DEV) / (R * P)
            if case["entropy"]:
                state["d_entropy"] = torch.full((R, P), 0.01 / (R * P), device=DEV)
            if case["top"]:
                state["d_top"] = torch.randn(R, P, case["top"], generator=g, device=DEV) / (R * P)
        return state
    N, H = case["tokens"], case["hidden"]
    if case["distinct"]:
        tokens = torch.arange(N, device=DEV)
    else:                                       # as in text: the r-th token in the share 1 / r
        tokens = (V ** torch.rand(N, generator=g, device=DEV, dtype=torch.float64) - 1).long().clamp_(max=V - 1)
    padding = None
    if case["padded"]:
        padding = V - 1
        tokens[torch.rand(N, generator=g, device=DEV) < case["padded"]] = padding
    table = torch.empty(V, H, dtype=dtype, device=DEV).normal_(0, 0.02, generator=g)
    state = dict(case=case, tokens=tokens, table=table, padding=padding)
    if kind == "table":
        table.requires_grad_()
        state["d_rows"] = torch.empty(N, H, dtype=dtype, device=DEV).normal_(0, 1e-3, generator=g)
    return state


# ----------------------------------------------------------------------------- plain forms

def _best(y, k):
    """Places of the k largest values of the last dimension, equal ones in their order."""
    bits = (y + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return ((key << 32) - torch.arange(y.shape[-1], device=DEV)).topk(k, dim=-1).indices


def _tell(s):
    case, tokens = s["case"], s["tokens"]
    y = s["logits"].detach().float()
    keep = tokens != IGNORED
    best = _best(y, case["top"]) if case["top"] else None
    if case["temperature"] != 1.0:
        y = y / case["temperature"]
    y = y - y.max(-1, keepdim=True).values
    e = y.exp()
    total = e.sum(-1, keepdim=True)
    y = y - total.log()
    out = dict(log_probs=torch.where(keep, y.gather(-1, tokens.clamp(min=0)[..., None])[..., 0], 0))
    p = e / total
    if case["entropy"]:
        entropy = -torch.where(p > 0, p * y, 0).sum(-1)
        out["entropy"] = torch.where(keep, entropy, 0)
    if best is not None:
        out["top_log_probs"] = torch.where(keep[..., None], y.gather(-1, best), 0)
        out["top_tokens"] = torch.where(keep[..., None], best, -1)
    if case["kind"] == "policy":
        rest = s["d_log_probs"] + s["d_top"].sum(-1) if case["top"] else s["d_log_probs"]
        d = p * rest[..., None]
        if case["entropy"]:
            d = d + p * torch.where(p > 0, y + entropy[..., None], 0) * s["d_entropy"][..., None]
        d = -d
        d.scatter_add_(-1, tokens.clamp(min=0)[..., None], s["d_log_probs"][..., None])
        if case["top"]:
            d.scatter_add_(-1, best, s["d_top"])
        out["d_logits"] = (torch.where(keep[..., None], d, 0) / case["temperature"]).to(s["logits"].dtype)
    return out


def _look_up(s):
    table, tokens, case = s["table"].detach(), s["tokens"], s["case"]
    out = dict(rows=(table[tokens].float() * case["scale"]).to(table.dtype))
    if case["kind"] == "table":
        d = torch.zeros(table.shape, dtype=torch.float32, device=DEV)
        d.index_add_(0, tokens, s["d_rows"].float() * case["scale"])
        if s["padding"] is not None:
            d[s["padding"]] = 0
        out["d_table"] = d.to(table.dtype)
    return out


# ----------------------------------------------------------------------------- the framework's calls

def _tell_own(s):
    from axonn_b200 import ops

    case = s["case"]
    r = ops.token_log_probs(s["logits"], s["tokens"], entropy=case["entropy"], top=case["top"], temperature=case["temperature"],
                            ignore_index=IGNORED)
    out = dict(log_probs=r.log_probs)
    if case["entropy"]:
        out["entropy"] = r.entropy
    if case["top"]:
        out["top_log_probs"], out["top_tokens"] = r.top_log_probs, r.top_tokens
    if case["kind"] == "policy":
        given = [(r.log_probs, s["d_log_probs"])]
        if case["entropy"]:
            given.append((r.entropy, s["d_entropy"]))
        if case["top"]:
            given.append((r.top_log_probs, s["d_top"]))
        out["d_logits"], = torch.autograd.grad([a for a, _ in given], [s["logits"]], [b for _, b in given])
    return out


def _look_up_own(s):
    from axonn_b200 import ops

    out = dict(rows=ops.embedding(s["tokens"], s["table"], scale=s["case"]["scale"], padding_idx=s["padding"]))
    if s["case"]["kind"] == "table":
        out["d_table"], = torch.autograd.grad([out["rows"]], [s["table"]], [s["d_rows"]])
    return out


def run(state):
    if state["case"]["kind"] in ("score", "policy"):
        return _tell_own(state) if own else _tell(state)
    return _look_up_own(state) if own else _look_up(state)


# ----------------------------------------------------------------------------- work, and the definition in 64 bits

def work(case):
    V, z = case["vocab"], SIZE[case["dtype"]]
    if case["kind"] in ("score", "policy"):
        count, kept, policy = case["rows"] * _positions(case), sum(_kept(case)), case["kind"] == "policy"
        told = count * (8 + 4 + 4 * case["entropy"] + 12 * case["top"])
        asked = count * (4 + 4 * case["entropy"] + 4 * case["top"]) if policy else 0
        return {"bytes": kept * V * z + policy * count * V * z + told + asked, "flops": kept * V * (4 + 2 * case["entropy"] + 6 * policy)}
    N, H = case["tokens"], case["hidden"]
    text = N * (1 - case["padded"])
    met = N if case["distinct"] else sum(1 - (1 - math.log1p(1 / r) / math.log(V)) ** text for r in range(1, V))      # different tokens
    bytes_ = N * 8 + met * H * z + N * H * z
    if case["kind"] == "table":
        bytes_ += N * H * z + V * H * z
    return {"bytes": bytes_, "flops": N * H * (2 if case["kind"] == "table" else 1)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("lookup", "table"):
        scale, table, tokens = float(case["scale"]), s["table"].detach(), s["tokens"]
        out = dict(rows=table.index_select(0, tokens).double().mul_(scale))
        if case["kind"] == "table":
            counts = torch.ones_like(tokens, dtype=torch.float64)
            if s["padding"] is not None:
                counts[tokens == s["padding"]] = 0
            out["d_table"] = torch.zeros(table.shape, dtype=torch.float64, device=DEV).index_add_(0, tokens, s["d_rows"].double() * counts[:, None], alpha=scale)
        return out
    tokens, T, V, P = s["tokens"].reshape(-1), float(case["temperature"]), case["vocab"], _positions(case)
    told = {k: [] for k in ("log_probs", "entropy", "top_log_probs", "d_logits")}
    flat = {k: s[k].reshape(tokens.numel(), -1) for k in ("d_log_probs", "d_entropy", "d_top") if k in s}
    step = max(1, (1 << 27) // V)
    for a in range(0, tokens.numel(), step):
        at = torch.arange(a, min(a + step, tokens.numel()), device=DEV)
        z = s["logits"].detach()[at // P, at % P].double() / T
        t = tokens[at]
        there = (t >= 0)[:, None].double()
        log_p = z - torch.logsumexp(z, -1, keepdim=True)
        hot = torch.zeros_like(z)
        hot[torch.arange(at.numel(), device=DEV), t.clamp(min=0)] = 1
        finite = log_p.masked_fill(log_p == -math.inf, 0)
        told["log_probs"].append(torch.where(t >= 0, (hot * finite).sum(-1), 0))
        p = log_p.exp()
        H = -(p * finite).sum(-1, keepdim=True)
        told["entropy"].append((H * there)[:, 0])
        if case["top"]:
            order = torch.sort(s["logits"].detach()[at // P, at % P].double(), dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            told["top_log_probs"].append(torch.where(there > 0, log_p.gather(1, order), 0))
        if case["kind"] == "policy":
            # d of sum_j c_j log p_j + h H by z: c - p sum c, and -h p (log p + H)
            c = hot * flat["d_log_probs"][at].double()
            if case["top"]:
                c.scatter_add_(1, order, flat["d_top"][at].double())
            d = c - p * c.sum(-1, keepdim=True)
            if case["entropy"]:
                d -= flat["d_entropy"][at].double() * p * (finite + H)
            told["d_logits"].append(d * there / T)
    shape = s["tokens"].shape
    out = dict(log_probs=torch.cat(told["log_probs"]).view(shape))
    if case["entropy"]:
        out["entropy"] = torch.cat(told["entropy"]).view(shape)
    if case["top"]:
        out["top_log_probs"], out["top_tokens"] = torch.cat(told["top_log_probs"]).view(*shape, -1), None
    if case["kind"] == "policy":
        out["d_logits"] = torch.cat(told["d_logits"]).view(*shape, V)
    return out
