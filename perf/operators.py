"""Generation with a block cache: the operators that a step of cached decoding and of beam search is made of.

A request's keys and values lie in blocks of ``block_tokens`` tokens, in 8 bits, with a power-of-two scale for each block
and KV head; a table names the blocks of every request.  A step plans the places of its new tokens (``plan_blocks``), stores
their keys and values (``store_blocks``), attends to everything that is stored (``cached_attention``) and, in beam search,
selects the continuations (``beam_select``) and lets the rows go on from their parents (``reorder_blocks``).

Sizes are those of the package's own configurations (GPT-1.3B: 16 heads of 128, 2048 positions, vocabulary 50304; Llama-8B:
32 query and 8 KV heads of 128, 4096 positions, vocabulary 128256; Mixtral: vocabulary 32000) and generic ones.
"""

import math

import torch

own = False
DEV = "cuda"
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LOWEST_EXPONENT = -100


def listed():
    return [
        # bookkeeping of one decoding step of a full batch: latency
        dict(name="plan_decode", kind="plan", requests=256, tokens=1, block_tokens=64, context=4096),
        # bookkeeping of a batch of prompts that enter the cache together
        dict(name="plan_prompts", kind="plan", requests=96, tokens=2048, block_tokens=64, context=0),
        # one decoding step of a Llama-8B layer: rotation, a token per request behind what its block holds
        dict(name="store_decode", kind="store", requests=128, tokens=1, block_tokens=64, context=1000, kv_heads=8, per_kv=4,
             head_dim=128, codes="e4m3", dtype="bf16", rope=True),
        # prompts of a GPT-1.3B layer (learned positions, no rotation), ragged lengths up to the model's
        dict(name="store_prompts", kind="store", requests=16, tokens=2048, block_tokens=64, context=0, kv_heads=16, per_kv=1,
             head_dim=128, codes="int8", dtype="bf16", rope=False),
        # one request, a short context: latency
        dict(name="attend_one_request", kind="attend", requests=1, tokens=1, shortest=900, context=900, block_tokens=64, kv_heads=8,
             per_kv=4, head_dim=128, codes="e4m3", dtype="bf16"),
        # a batch of requests of very different lengths, Llama-8B heads
        dict(name="attend_ragged_batch", kind="attend", requests=64, tokens=1, shortest=17, context=8192, block_tokens=64, kv_heads=8,
             per_kv=4, head_dim=128, codes="e4m3", dtype="bf16"),
        # long documents: few requests, many tokens each
        dict(name="attend_long_context", kind="attend", requests=3, tokens=1, shortest=60001, context=131072, block_tokens=128,
             kv_heads=8, per_kv=4, head_dim=128, codes="e4m3", dtype="fp16"),
        # several new tokens per request (a prompt that goes on, drafted tokens), GPT-1.3B heads
        dict(name="attend_new_tokens", kind="attend", requests=24, tokens=8, shortest=700, context=2048, block_tokens=32,
             kv_heads=16, per_kv=1, head_dim=128, codes="int8", dtype="bf16"),
        # one prompt, four beams, Mixtral's vocabulary: latency
        dict(name="select_one_prompt", kind="select", groups=1, beams=4, vocab=32000, dtype="bf16", ended=False),
        # a batch of prompts over Llama-8B's vocabulary, some beams have ended
        dict(name="select_batch", kind="select", groups=32, beams=8, vocab=128256, dtype="bf16", ended=True),
        # four beams of one prompt through the cache of a GPT-1.3B model
        dict(name="reorder_one_prompt", kind="reorder", layers=24, groups=1, beams=4, width=8, block_tokens=64, kv_heads=16,
             head_dim=128, codes="e4m3"),
        # a batch of prompts through the cache of a Llama-8B model
        dict(name="reorder_batch", kind="reorder", layers=32, groups=16, beams=4, width=8, block_tokens=64, kv_heads=8,
             head_dim=128, codes="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "store", "attend", "attend", "select", "reorder"])
    blocks = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        tokens = _log(rng, 1, 2048)
        requests = _log(rng, 1, max(1, min(2048, 196608 // tokens)))
        return dict(kind=kind, requests=requests, tokens=tokens, block_tokens=blocks, context=rng.choice([0, _log(rng, 1, 8192)]))
    codes, head_dim, dtype = rng.choice(["e4m3", "int8"]), rng.choice([64, 128]), rng.choice(["bf16", "fp16"])
    kv_heads, per_kv = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 3, 4, 8])
    if kind == "store":
        tokens = _log(rng, 1, 2048)
        requests = _log(rng, 1, max(1, min(512, 65536 // (tokens * kv_heads * max(1, per_kv // 2)))))
        return dict(kind=kind, requests=requests, tokens=tokens, block_tokens=blocks, context=rng.choice([0, _log(rng, 1, 2000)]),
                    kv_heads=kv_heads, per_kv=per_kv, head_dim=head_dim, codes=codes, dtype=dtype, rope=rng.random() < 0.7)
    if kind == "attend":
        tokens = rng.choice([1, 1, 1, 1, 2, 3, 5, 8, 17])
        context = _log(rng, tokens, 65536)
        requests = _log(rng, 1, max(1, min(256, 2250000 // (context * kv_heads * -(-tokens * per_kv // 8)))))
        return dict(kind=kind, requests=requests, tokens=tokens, shortest=max(tokens, int(context * rng.uniform(0.02, 1))), context=context,
                    block_tokens=blocks, kv_heads=kv_heads, per_kv=per_kv, head_dim=head_dim, codes=codes, dtype=dtype)
    if kind == "select":
        beams, vocab, dtype = rng.randint(1, 16), _log(rng, 1000, 131072), rng.choice(["bf16", "bf16", "fp16", "fp32"])
        groups = _log(rng, 1, max(1, min(64, (15000000 if dtype == "fp32" else 30000000) // (beams * vocab))))
        return dict(kind=kind, groups=groups, beams=beams, vocab=vocab, dtype=dtype, ended=rng.random() < 0.5)
    layers, beams = _log(rng, 1, 32), rng.randint(2, 8)
    groups = _log(rng, 1, max(1, 1024 // (layers * beams)))
    return dict(kind=kind, layers=layers, groups=groups, beams=beams, width=rng.randint(1, 8), block_tokens=blocks,
                kv_heads=rng.choice([1, 2, 4, 8]), head_dim=head_dim, codes=codes)


# ----------------------------------------------------------------------------- inputs

def _lengths(case):
    """Tokens of every request, a function of the case alone: evenly spread between the shortest and the longest."""
    R, lo, hi = case["requests"], case["shortest"], case["context"]
    return [hi if R == 1 else lo + (hi - lo) * i // (R - 1) for i in range(R)]


def _spread(case):
    """Lengths before and new tokens of every request of a plan or store case."""
    R, S, ctx = case["requests"], case["tokens"], case["context"]
    before = [ctx * (i % 7 + 1) // 7 + (i * 13) % 50 * (ctx > 0) for i in range(R)]
    return before, [S - (S // 2) * (i % 5) // 4 for i in range(R)]


def _order(n, g):
    return torch.randperm(n, generator=g, device=DEV)


def _codes(case, blocks, g):
    """Keys or values as the cache holds them: normal values in 8 bits, and the scales of blocks of different sizes."""
    G, BT, D = case["kv_heads"], case["block_tokens"], case["head_dim"]
    out = torch.empty(blocks, G, BT, D, dtype=CODES[case["codes"]], device=DEV)
    chunk = max(1, (1 << 26) // (G * BT * D))
    for a in range(0, blocks, chunk):
        x = torch.randn(min(chunk, blocks - a), G, BT, D, generator=g, device=DEV)
        out[a:a + chunk] = (x * 80).clamp_(-448, 448).to(out.dtype) if case["codes"] == "e4m3" else (x * 30).round_().clamp_(-127, 127).to(out.dtype)
    at = -6.0 if case["codes"] == "e4m3" else -5.0
    return out, torch.exp2(at + torch.randint(-1, 2, (blocks, G), generator=g, device=DEV))


def _filled_tables(lengths, width, BT, ids):
    """Tables whose rows name the blocks of ``lengths`` tokens, taken from ``ids`` in turn; -1 behind them."""
    held = (lengths + BT - 1) // BT
    col = torch.arange(width, device=DEV)
    at = (held.cumsum(0) - held)[:, None] + col
    return torch.where(col < held[:, None], ids[at.clamp(max=ids.numel() - 1)], -1).int()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    if kind == "select":
        B, K, V = case["groups"], case["beams"], case["vocab"]
        logits = (torch.randn(B, K, V, generator=g, device=DEV) * 2.5).to(TYPES[case["dtype"]])
        scores = -20 * torch.rand(B, K, generator=g, device=DEV)
        done = torch.rand(B, K, generator=g, device=DEV) < 0.2 if case["ended"] else None
        return dict(case=case, logits=logits, scores=scores, done=done, eos=V // 3 if case["ended"] else None)
    BT = case["block_tokens"]
    if kind == "reorder":
        L, B, K, W = case["layers"], case["groups"], case["beams"], case["width"]
        R = B * K
        N = R * (W + 1)
        ids = _order(N, g).int()
        k, ks = _codes(case, L * N, g)
        v, vs = _codes(case, L * N, g)
        stacked = [t.view(L, N, *t.shape[1:]) for t in (k, v, ks, vs)]
        # every group has written its own share of its last block; every row of a group moves on but the first
        length = [(W - 1) * BT + BT * (i % 4 * 2 + 1) // 8 for i in range(B)]
        lengths = torch.tensor(length, dtype=torch.int32, device=DEV).repeat_interleave(K)
        parents = (torch.randint(1, K, (B, K), generator=g, device=DEV) + torch.arange(K, device=DEV)) % K
        parents[:, 0] = 0
        return dict(case=case, blocks=stacked, tables=ids[:R * W].view(R, W), lengths=lengths, spare=ids[R * W:], parents=parents.int())
    if kind == "attend":
        lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)[_order(case["requests"], g)]
        width = -(-case["context"] // BT)
        blocks = sum(-(-n // BT) for n in _lengths(case))
        k, ks = _codes(case, blocks, g)
        v, vs = _codes(case, blocks, g)
        tables = _filled_tables(lengths, width, BT, _order(blocks, g))
        q = (2 * torch.randn(case["requests"], case["tokens"], case["kv_heads"] * case["per_kv"], case["head_dim"], generator=g,
                             device=DEV)).to(TYPES[case["dtype"]])
        return dict(case=case, q=q, blocks=[k, v, ks, vs], tables=tables, lengths=lengths)
    before, new = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in _spread(case))
    order = _order(case["requests"], g)
    before, new = before[order], new[order]
    width = (max(_spread(case)[0]) + case["tokens"] + BT - 1) // BT
    held = sum(-(-n // BT) for n in _spread(case)[0])
    total = sum(-(-(n + m) // BT) + 1 for n, m in zip(*_spread(case)))
    free = _order(total, g).int()
    tables = _filled_tables(before, width, BT, free)
    taken = torch.full((1,), held, dtype=torch.int32, device=DEV)
    plan = dict(case=case, lengths=before, new=new, tables=tables, free=free, taken=taken)
    if kind == "plan":
        return plan
    placed = _plan(plan)
    G, P, D = case["kv_heads"], case["per_kv"], case["head_dim"]
    k, ks = _codes(case, total, g)
    v, vs = _codes(case, total, g)
    qkv = torch.randn(case["requests"], case["tokens"], G, P + 2, D, generator=g, device=DEV) * (1 + 2 * torch.rand(D, generator=g, device=DEV))
    table = None
    if case["rope"]:
        angle = torch.outer(torch.arange(width * BT, device=DEV, dtype=torch.float64),
                            500000.0 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D))
        table = torch.stack([angle.cos(), angle.sin()], -1).float()
    return dict(case=case, qkv=qkv.to(TYPES[case["dtype"]]), blocks=[k, v, ks, vs], slots=placed["slots"], positions=placed["positions"],
                table=table)


# ----------------------------------------------------------------------------- plain forms

def _plan(s):
    lengths, new, free, S, BT = s["lengths"].long(), s["new"].long(), s["free"], s["case"]["tokens"], s["case"]["block_tokens"]
    W, N = s["tables"].shape[1], free.numel()
    held = (lengths + BT - 1) // BT
    need = ((lengths + new + BT - 1) // BT).clamp(max=W) - held
    base = s["taken"] + need.cumsum(0) - need
    got = torch.minimum((N - base).clamp(min=0), need)
    after = torch.minimum(lengths + new, (held + got) * BT)
    col = torch.arange(W, device=DEV) - held[:, None]
    fresh = (col >= 0) & (col < got[:, None])
    tables = torch.where(fresh, free[(base[:, None] + col).clamp(0, N - 1)], s["tables"])
    step = torch.arange(S, device=DEV)
    at = lengths[:, None] + step
    block = tables.long().gather(1, (at // BT).clamp(max=W - 1))
    there = step < (after - lengths)[:, None]
    return dict(slots=torch.where(there, block * BT + at % BT, -1), positions=torch.where(there, at, -1).int(), lengths=after.int(),
                taken=(s["taken"] + got.sum()).int(), tables=tables)


def _exponent(largest, codes):
    """The least e with largest <= M 2^e, M the largest code; at least LOWEST_EXPONENT."""
    m, e = torch.frexp(largest)                       # largest = 2 m 2^(e - 1), 1 <= 2 m < 2
    top = int(math.log2(LARGEST[codes]))
    e = e - 1 - top + (2 * m > LARGEST[codes] / 2 ** top)
    return torch.where(largest > 0, e, LOWEST_EXPONENT).clamp(min=LOWEST_EXPONENT)


def _power(e):
    """2^e to the bit, from the exponent field of a 32-bit number."""
    return ((e + 127) << 23).int().view(torch.float32)


def _to_codes(x, codes):
    return x.to(torch.float8_e4m3fn) if codes == "e4m3" else x.round().to(torch.int8)


def _rotate(x, table, positions):
    """Pairs (i, i + D / 2) of the heads of ``x [R, S, ..., D]`` by the angles of their positions."""
    h = x.shape[-1] // 2
    cs = table[positions.clamp(min=0).long()].view(*x.shape[:2], *[1] * (x.ndim - 3), h, 2)
    a, b, cos, sin = x[..., :h], x[..., h:], cs[..., 0], cs[..., 1]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _store(s):
    qkv, (k, v, ks, vs), slots, codes = s["qkv"], s["blocks"], s["slots"], s["case"]["codes"]
    R, S, G, _, D = qkv.shape
    N, BT = k.shape[0], k.shape[2]
    q = qkv[:, :, :, :-2]
    if s["table"] is not None:
        q = _rotate(q.float(), s["table"], s["positions"])
        q = torch.where(slots.view(R, S, 1, 1, 1) >= 0, q, 0).to(qkv.dtype)
    there = slots.reshape(-1) >= 0
    block = torch.where(there, slots.reshape(-1) // BT, N)          # block N takes what has no place
    within = torch.where(there, slots.reshape(-1) % BT, 0)
    first = torch.full((N + 1,), BT, device=DEV).scatter_reduce_(0, block, within, "amin")[:N, None]
    row_block = slots[:, 0] // BT                                   # the block of a row that may hold tokens already
    for x, c, scale in ((qkv[:, :, :, -2], k, ks), (qkv[:, :, :, -1], v, vs)):
        x = x.float()
        if s["table"] is not None and c is k:
            x = _rotate(x, s["table"], s["positions"])
        x = x.reshape(R * S, G, D)
        largest = torch.zeros(N + 1, G, device=DEV).scatter_reduce_(0, block[:, None].expand(-1, G), x.abs().amax(-1), "amax")[:N]
        new = _power(_exponent(largest, codes))
        old = scale.clone()
        scale.copy_(torch.where(first == BT, old, torch.where(first > 0, torch.maximum(new, old), new)))
        shrink = (old[row_block] / scale[row_block])[..., None, None]
        held = (torch.arange(BT, device=DEV) < first[row_block])[:, None, :, None]
        c[row_block] = _to_codes(torch.where(held, c[row_block].float() * shrink, c[row_block].float()), codes)
        wide = torch.cat([scale, scale[:1]])[block][..., None]
        coded = _to_codes(torch.where(there[:, None, None], x / wide, 0), codes)
        # what has no place goes behind the cache
        flat = torch.cat([c.view(torch.uint8), torch.empty_like(c[:1]).view(torch.uint8)]).transpose(1, 2).reshape((N + 1) * BT, G, D)
        flat[block * BT + within] = coded.view(torch.uint8)
        c.view(torch.uint8).copy_(flat[:N * BT].view(N, BT, G, D).transpose(1, 2))
    return [q.reshape(R, S, -1, D) if s["table"] is not None else None, k, v, ks, vs]


def _attend(s):
    q, (k, v, ks, vs), tables, lengths = s["q"], s["blocks"], s["tables"].long(), s["lengths"].long()
    R, S, H, D = q.shape
    W, (G, BT) = tables.shape[1], k.shape[1:3]
    at = tables.clamp(min=0)
    keys, values = ((c[at].float() * sc[at][..., None, None]).transpose(2, 3).reshape(R, W * BT, G, D) for c, sc in ((k, ks), (v, vs)))
    qs = q.float().view(R, S, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(R, G, -1, D)
    scores = qs @ keys.permute(0, 2, 3, 1) / math.sqrt(D)
    last = lengths[:, None] - S + torch.arange(S, device=DEV)       # the token that a query stands at is the last that it sees
    seen = (torch.arange(W * BT, device=DEV) <= last[..., None]).repeat_interleave(H // G, 1)[:, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    values = torch.where((torch.arange(W * BT, device=DEV) < lengths[:, None])[..., None, None], values, 0)
    o = p @ values.transpose(1, 2) / p.sum(-1, keepdim=True)
    o = o.view(R, G, S, H // G, D).permute(0, 2, 1, 3, 4).reshape(R, S, H, D)
    return o.to(q.dtype)


def _select(s):
    x, scores, done, eos = s["logits"].double(), s["scores"], s["done"], s["eos"]
    B, K, V = x.shape
    top = x.amax(-1, keepdim=True)
    value = scores.double()[..., None] + (x - top) - (x - top).exp().sum(-1, keepdim=True).log()
    if done is not None:
        ending = torch.where(torch.arange(V, device=DEV) == eos, scores.double()[..., None], float("-inf"))
        value = torch.where(done[..., None], ending, value)
    value = value.masked_fill(value.isnan(), float("-inf")).view(B, K * V)
    value, at = value.sort(stable=True, dim=-1, descending=True)        # equal values in the order of their indices
    value, at = value[:, :K], at[:, :K]
    parents, tokens = at // V, at % V
    ended = None if done is None else done.gather(1, parents) | (tokens == eos)
    return [value.float(), tokens, parents.int(), ended]


def _reorder(s):
    k, v, ks, vs = s["blocks"]
    tables, lengths, spare, parents = s["tables"], s["lengths"], s["spare"], s["parents"]
    R, BT = tables.shape[0], k.shape[3]
    row = torch.arange(R, device=DEV)
    parent = row // parents.shape[1] * parents.shape[1] + parents.view(-1)
    length = lengths[parent]
    part = length % BT
    current = (length // BT).clamp(max=tables.shape[1] - 1).long()
    moved = (parent != row) & (part > 0)
    source = torch.where(moved, tables[parent, current], spare).long()
    target = spare.long()
    keep = (torch.arange(BT, device=DEV) < part[:, None])[:, None, :, None] & moved[:, None, None, None]
    for c, scale in ((k, ks), (v, vs)):
        raw = c.view(torch.uint8)
        raw[:, target] = torch.where(keep, raw[:, source], raw[:, target])
        scale[:, target] = scale[:, source]
    out = tables[parent]
    out[row, current] = torch.where(moved, spare, out[row, current])
    return [out, length, torch.where(moved, tables[row, current], spare), k, v, ks, vs]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        if kind == "plan":
            p = _plan(state)
            state["tables"].copy_(p["tables"])
            return [p["slots"], p["positions"], p["lengths"], p["taken"], state["tables"]]
        return {"store": _store, "attend": _attend, "select": _select, "reorder": _reorder}[kind](state)
    from axonn_b200 import ops

    if kind == "plan":
        p = ops.plan_blocks(state["lengths"], state["new"], state["tables"], state["free"], state["taken"], state["case"]["tokens"],
                            state["case"]["block_tokens"])
        return [p.slots, p.positions, p.lengths, p.taken, state["tables"]]
    if kind == "store":
        layer = ops.BlockLayer(*state["blocks"])
        q = ops.store_blocks(state["qkv"], layer, state["slots"], state["positions"], state["table"])
        return [q, *layer]      # the cache as it is kept, codes beside their scales: both are the same to the bit in every form
    if kind == "attend":
        return ops.cached_attention(state["q"], ops.BlockLayer(*state["blocks"]), state["tables"], state["lengths"])
    if kind == "select":
        step = ops.beam_select(state["logits"], state["scores"], state["done"], state["eos"])
        return list(step)
    blocks = ops.BlockLayer(*state["blocks"])
    return [*ops.reorder_blocks(blocks, state["tables"], state["lengths"], state["spare"], state["parents"]), *blocks]


# ----------------------------------------------------------------------------- work and 64 bits

def work(case):
    kind = case["kind"]
    if kind == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + 32 * case["groups"] * case["beams"], "flops": 4 * n}
    BT = case["block_tokens"]
    if kind == "reorder":
        part = [BT * (i % 4 * 2 + 1) // 8 for i in range(case["groups"])]
        moved = sum(p * (case["beams"] - 1) for p in part if p)
        rows = case["groups"] * case["beams"]
        return {"bytes": 4 * moved * case["layers"] * case["kv_heads"] * case["head_dim"] + 8 * rows * (case["width"] + 2), "flops": 0}
    if kind == "plan":
        before, new = _spread(case)
        fresh = sum(-(-(n + m) // BT) - -(-n // BT) for n, m in zip(before, new))
        return {"bytes": 12 * case["requests"] * case["tokens"] + 12 * case["requests"] + 8 * fresh, "flops": 0}
    G, P, D = case["kv_heads"], case["per_kv"], case["head_dim"]
    if kind == "store":
        tokens = sum(_spread(case)[1])
        rope = case["rope"]
        q = 2 * G * P * D * (tokens + case["requests"] * case["tokens"]) if rope else 0
        angles = 4 * D * min(tokens, max(map(sum, zip(*_spread(case))))) if rope else 0
        return {"bytes": tokens * (6 * G * D + 12) + q + angles, "flops": tokens * G * (P + 1) * 3 * D if rope else 0}
    seen = sum(_lengths(case))
    q = 4 * case["requests"] * case["tokens"] * G * P * D
    return {"bytes": 2 * seen * G * D + 8 * G * seen // BT + 4 * seen // BT + q, "flops": 4 * seen * case["tokens"] * G * P * D}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return None
    if kind == "select":
        x = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
        if s["done"] is not None:
            x[s["done"]] = float("-inf")
            x[..., s["eos"]] = torch.where(s["done"], s["scores"].double(), x[..., s["eos"]])
        return [x.flatten(1).topk(case["beams"], -1)[0], None, None, None]
    if kind == "reorder":
        # copies: the caches as they are afterwards, row by row
        caches, K, BT = s["blocks"], case["beams"], case["block_tokens"]
        tables, spare, lengths = s["tables"].tolist(), s["spare"].tolist(), s["lengths"].tolist()
        before = [c.clone() for c in caches]
        for r, j in enumerate(s["parents"].flatten().tolist()):
            parent = r // K * K + j
            full, part = divmod(lengths[parent], BT)
            if parent != r and part:
                for c, b in zip(caches[:2], before[:2]):
                    c[:, spare[r], :, :part] = b[:, tables[parent][full], :, :part]
                for c, b in zip(caches[2:], before[2:]):
                    c[:, spare[r]] = b[:, tables[parent][full]]
        return [None, None, None, *caches]
    if kind == "store":
        return _store_exactly(s)
    return _attend_exactly(s)


def _store_exactly(s):
    """Request by request, block by block; the angles are those of the table that the call is given."""
    case, qkv, slots = s["case"], s["qkv"].double(), s["slots"].tolist()
    BT, codes, (R, S, G, _, D) = case["block_tokens"], case["codes"], qkv.shape
    if R * (S + BT) / BT > 3000:
        return None
    q = None
    if s["table"] is not None:
        turn = torch.view_as_complex(s["table"].double())[s["positions"].clamp(min=0).long()][:, :, None, None]
        z = torch.complex(qkv[..., :D // 2], qkv[..., D // 2:]) * turn
        rotated = torch.cat([z.real, z.imag], -1)
        q = rotated[:, :, :, :-2].reshape(R, S, -1, D) * (s["slots"] >= 0)[..., None, None]
        qkv = torch.cat([rotated[:, :, :, :-1], qkv[:, :, :, -1:]], 3)
    k, v, ks, vs = s["blocks"]
    for r in range(R):
        i = 0
        while i < S and slots[r][i] >= 0:
            block, at = divmod(slots[r][i], BT)
            n = min(BT - at, sum(t >= 0 for t in slots[r][i:i + BT - at]))
            for c, scale, x in ((k, ks, qkv[r, i:i + n, :, -2]), (v, vs, qkv[r, i:i + n, :, -1])):
                x = x.transpose(0, 1)
                half, e = torch.frexp(x.abs().amax((1, 2)) / LARGEST[codes])      # half 2^e, half in [0.5, 1)
                power = torch.where(half == 0.5, 0.5, 1.0) * 2.0 ** e.clamp(min=-200).double()
                power = power.clamp(min=2.0 ** LOWEST_EXPONENT)
                if at:
                    power = torch.maximum(power, scale[block].double())
                    old = c[block, :, :at].double() * (scale[block].double() / power)[:, None, None]
                    c[block, :, :at] = _to_codes(old, codes)
                scale[block] = power.float()
                c[block, :, at:at + n] = _to_codes(x / power[:, None, None], codes)
            i += n
    return [q, k, v, ks, vs]


def _attend_exactly(s):
    """Request by request over its own tokens."""
    case, (k, v, ks, vs) = s["case"], s["blocks"]
    R, S, H, D = s["q"].shape
    G, BT = case["kv_heads"], case["block_tokens"]
    out = []
    for r, n in enumerate(s["lengths"].tolist()):
        ids = s["tables"][r, :(n + BT - 1) // BT].long()
        K, V = ((c[ids].double() * sc[ids].double()[..., None, None]).transpose(1, 2).reshape(-1, G, D)[:n] for c, sc in ((k, ks), (v, vs)))
        q = s["q"][r].double().view(S, G, H // G, D)
        a = torch.einsum("sgpd,tgd->gpst", q, K) * D ** -0.5
        late = torch.arange(n, device=DEV) > torch.arange(n - S, n, device=DEV)[:, None]
        p = a.masked_fill(late, float("-inf")).softmax(-1)
        out.append(torch.einsum("gpst,tgd->sgpd", p, V).reshape(S, H, D))
    return torch.stack(out)
