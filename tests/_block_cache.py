"""Inputs and 64-bit oracles of the block cache's tests, written from the definitions, request by request."""



import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def as_codes(x, dtype):
    return x.clamp(-448, 448).to(dtype) if dtype == E4M3 else x.round().clamp(-127, 127).to(dtype)


def make_cache(blocks, G, BT, D, dtype, seed=0, spread=1):
    """Codes of normal values, scales of powers of two within ``spread`` octaves around 2^-6."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn(blocks, G, BT, D, generator=g) * (64 if dtype == E4M3 else 32)
        out.append(as_codes(x, dtype))
    scales = [torch.exp2(-6.0 + torch.randint(-spread, spread + 1, (blocks, G), generator=g)).float() for _ in range(2)]
    return out[0], out[1], scales[0], scales[1]


def make_tables(lengths, W, BT, blocks, seed=0):
    """Every request's blocks, drawn without repetition; -1 behind them."""
    ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    tables = torch.full((len(lengths), W), -1, dtype=torch.int32)
    for r, n in enumerate(lengths):
        for i in range(-(-n // BT)):
            tables[r, i] = ids.pop()
    return tables


def attend64(q, layer, tables, lengths, new=None, scale=None):
    """(outputs, sums of p |v|) in 64 bits; ``q [R, S, H, D]``."""
    k, v, ks, vs = layer
    R, S, H, D = q.shape
    G, BT = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    out, size = torch.zeros(R, S, H, D, dtype=torch.float64), torch.zeros(R, S, H, D, dtype=torch.float64)
    for r, n in enumerate(lengths):
        m = S if new is None else min(new[r], S)
        token = torch.arange(min(n, tables.shape[1] * BT))
        block = tables[r].long()[token // BT]
        token, block = (x[(block >= 0) & (block < k.shape[0])] for x in (token, block))
        for g in range(G):
            h = slice(g * H // G, (g + 1) * H // G)
            K = k.float()[block, g, token % BT].double() * ks[block, g].double()[:, None]
            V = v.float()[block, g, token % BT].double() * vs[block, g].double()[:, None]
            for i in range(m):
                seen = int((token < n - m + i + 1).sum())
                if seen:
                    p = (q[r, i, h].double() @ K[:seen].T * scale).softmax(-1)
                    out[r, i, h], size[r, i, h] = p @ V[:seen], p @ V[:seen].abs()
    return out, size


def store64(qkv, cache, slots, positions=None, table=None):
    """The cache (k, v, k_scale, v_scale) after the store, and the rotated queries in 64 bits."""
    R, S, G, n, D = qkv.shape
    x = qkv.double().clone()
    q = None
    there = slots >= 0
    if table is not None:
        there = there & (positions >= 0) & (positions < len(table))
        h = D // 2
        # 32-bit products, as documented: what is rounded decides at borders of the codes
        y = qkv.float()
        cs = table[positions.clamp(0, len(table) - 1).long()][:, :, None, None]
        a, b, c, s = y[..., :h], y[..., h:], cs[..., 0], cs[..., 1]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1).double()
        x[:, :, :, :-1] = turned[:, :, :, :-1]
        wide = qkv.double()
        a, b, c, s = wide[..., :h], wide[..., h:], c.double(), s.double()
        q = torch.cat([a * c - b * s, b * c + a * s], -1)[:, :, :, :-2].reshape(R, S, -1, D) * there[..., None, None]
    out = [t.clone() for t in cache]
    BT = cache[0].shape[2]
    by_block = {}
    for r in range(R):
        for i in range(S):
            if there[r, i]:
                by_block.setdefault(int(slots[r, i]) // BT, []).append((r, i, int(slots[r, i]) % BT))
    for b, tokens in by_block.items():
        held = min(t for _, _, t in tokens)
        for which in (0, 1):
            codes, scales = out[which], out[2 + which]
            most = LARGEST[codes.dtype]
            for g in range(G):
                new = torch.stack([x[r, i, g, which - 2] for r, i, _ in tokens])
                size = new[new.isfinite()].abs().max().item() if new.isfinite().any() else 0.0
                e = -100
                while size > most * 2.0 ** e:
                    e += 1
                scale = 2.0 ** e
                if held:
                    old = float(scales[b, g])
                    scale = max(scale, old)
                    if scale > old:
                        moved = codes[b, g, :held].double() * (old / scale)
                        put(codes, (b, g, slice(0, held)), code64(moved, codes.dtype))
                scales[b, g] = scale
                for j, (_, _, t) in enumerate(tokens):
                    put(codes, (b, g, t), code64(new[j] / scale, codes.dtype))
    return out, q


def code64(x, dtype):
    if dtype == INT8:
        return torch.where(x.isnan(), 0, x).clamp(-127, 127).round().to(dtype)
    return x.clamp(-448, 448).to(torch.float32).to(dtype)


def put(codes, at, value):
    codes.view(torch.uint8)[at] = value.view(torch.uint8)


def same_bits(a, b):
    if a.numel() == 0:
        return a.dtype == b.dtype and a.shape == b.shape
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def attend_bound(out64, size64, dtype):
    """Rounding of the result (half a step); probabilities are rounded to fp16 (2^-11 of each), and scores of at most ten, the sums of
    128 products of 32 bits, are off by 128 x 10 x 2^-24 = 2^-13.7, which moves numerator and denominator by at most 0.7 of that."""
    return torch.finfo(dtype).eps / 2 * out64.abs() + (2.0 ** -11 + 2.0 ** -13) * size64 * (1 + torch.finfo(dtype).eps)


def rope_table(n, D, theta=10000.0):
    angle = torch.outer(torch.arange(n, dtype=torch.float64), theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    return torch.stack([angle.cos(), angle.sin()], -1).float()


