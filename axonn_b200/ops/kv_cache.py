"""Key/value cache in blocks of 8-bit codes: planning, storing, attending and reordering (``csrc/kv_cache.cu``,
``csrc/cached_attention.cu``).

One layer of a cache is a ``BlockLayer``: codes ``[blocks, kv_heads, block_tokens, D]`` (``torch.float8_e4m3fn`` or
``torch.int8``) and fp32 scales ``[blocks, kv_heads]``, powers of two; a value is its code times the scale of its block
and head.  ``tables [R, W]`` (int32) names the blocks of every request in order, -1 behind them, and ``lengths [R]``
(int32) says how many tokens they hold.  ``models.BlockCache`` keeps all of these for a model; the functions here take
them as tensors, never synchronise and can be captured into a CUDA graph.  They belong to inference: a tensor that
requires a gradient is refused.

The reference has no cache of its own: its patched Hugging Face models bring theirs
(``axonn/models/transformers/modify_llama.py``).
"""

import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from .direct import host_paths

BLOCK_TOKENS = (16, 32, 64, 128)
CODE_TYPES = (torch.float8_e4m3fn, torch.int8)
LOWEST_EXPONENT = -100          # of a scale: values below 2^-100 of a block without larger ones are zeros
_HALF = {torch.bfloat16: 0, torch.float16: 1}


class BlockLayer(NamedTuple):
    """Codes and scales of one layer (of several, stacked in front, for ``reorder_blocks``)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class BlockPlan(NamedTuple):
    """Places of new tokens: ``slots [R, S]`` (int64, ``block * block_tokens + place``), ``positions [R, S]`` (int32), both -1 for
    a token without a place, and the requests' ``lengths [R]`` and the blocks ``taken [1]`` afterwards (int32)."""

    slots: torch.Tensor
    positions: torch.Tensor
    lengths: torch.Tensor
    taken: torch.Tensor


def _int32(name, t, *shape):
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a dense int32 tensor of shape {list(shape)}, not {t.dtype} {list(t.shape)}")


def _together(device, *tensors):
    """All tensors on one device, none with a gradient to be had."""
    for t in tensors:
        if t is not None:
            if t.device != device:
                raise ValueError(f"tensors on {device} and {t.device}")
            if t.requires_grad and torch.is_grad_enabled():
                raise RuntimeError("operations on the block cache have no derivative: call them under torch.no_grad()")


def _elsewhere(device):
    """Is ``device`` a GPU other than the current one?"""
    return device.type == "cuda" and device.index != torch._C._cuda_getDevice()


def _check_layer(layer, dims):
    k, v, ks, vs = layer
    if k.dtype not in CODE_TYPES or v.dtype != k.dtype:
        raise TypeError(f"codes are float8_e4m3fn or int8, both alike, not {k.dtype} and {v.dtype}")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError("scales are fp32")
    if k.ndim != dims or v.shape != k.shape or ks.shape != k.shape[:-2] or vs.shape != k.shape[:-2]:
        raise ValueError(f"codes {list(k.shape)} and {list(v.shape)} do not go with scales {list(ks.shape)} and {list(vs.shape)}")
    if k.shape[-2] not in BLOCK_TOKENS:
        raise ValueError(f"blocks hold 16, 32, 64 or 128 tokens, not {k.shape[-2]}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("the tensors of a block cache are dense")
    if k.is_cuda and (k.data_ptr() | v.data_ptr()) % 16:
        raise ValueError("the codes of a block cache start on 16 bytes")


def plan_blocks(lengths, new, tables, free, taken, tokens, block_tokens):
    """Places for the first ``new[r]`` of ``tokens`` tokens behind the ``lengths[r]`` that request ``r`` has (all int32).

    The blocks that are missing are the next ones of the list ``free``, of which ``taken[0]`` have been used, in the order of
    the requests; their ids are written into ``tables`` (in place: entries behind what a request holds).  A request whose row of
    the table is full, or that comes when the list is used up, gets places for as many tokens as there is room for: its
    ``lengths`` entry of the plan tells.  Tokens of an unfinished block that the table lacks (-1 within the length) are counted, but have no
    slot.  ``lengths`` and ``taken`` themselves are left as they are (numbers below 0 and beyond the
    list count as 0 and its end)."""
    if lengths.is_cuda and (host := host_paths()) is not None:
        out = host.plan_blocks(lengths, new, tables, free, taken, tokens, block_tokens)
        if out is not None:
            return BlockPlan(*out)
    dev, R = lengths.device, lengths.shape[0] if lengths.ndim == 1 else -1
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return plan_blocks(lengths, new, tables, free, taken, tokens, block_tokens)
    if block_tokens not in BLOCK_TOKENS:
        raise ValueError(f"blocks hold 16, 32, 64 or 128 tokens, not {block_tokens}")
    if tables.ndim != 2 or free.ndim != 1 or free.numel() == 0 or tables.shape[1] == 0 or tokens < 0:
        raise ValueError("plan_blocks takes lengths [R], new [R], tables [R, W], free [N], taken [1] and a number of tokens")
    _int32("lengths", lengths, R)
    _int32("new", new, R)
    _int32("tables", tables, R, tables.shape[1])
    _int32("free", free, free.shape[0])
    _int32("taken", taken, 1)
    if tables.shape[1] * block_tokens >= 1 << 31:
        raise ValueError(f"a row of {tables.shape[1]} blocks holds more than 2^31 - 1 tokens")
    _together(dev, new, tables, free, taken)
    if R == 0 or tokens == 0:
        return BlockPlan(torch.empty(R, tokens, dtype=torch.int64, device=dev), torch.empty(R, tokens, dtype=torch.int32, device=dev),
                         lengths.clone(), taken.clone())
    if not lengths.is_cuda:
        return _plan_torch(lengths, new, tables, free, taken, tokens, block_tokens)
    slots = torch.empty(R, tokens, dtype=torch.int64, device=dev)
    positions = torch.empty(R, tokens, dtype=torch.int32, device=dev)
    after, used = torch.empty_like(lengths), torch.empty_like(taken)
    st = _lib.lib().axb_plan_blocks(lengths.data_ptr(), new.data_ptr(), tables.data_ptr(), free.data_ptr(), taken.data_ptr(),
                                    slots.data_ptr(), positions.data_ptr(), after.data_ptr(), used.data_ptr(), R, tokens,
                                    tables.shape[1], free.shape[0], block_tokens, _lib.stream())
    _lib.check(st, "axb_plan_blocks")
    return BlockPlan(slots, positions, after, used)


def _plan_torch(lengths, new, tables, free, taken, S, BT):
    W, N = tables.shape[1], free.numel()
    length, add = lengths.long().clamp(min=0), new.long().clamp(0, S)
    held = ((length + BT - 1) // BT).clamp(max=W)
    need = ((length + add + BT - 1) // BT).clamp(max=W) - held
    taken = taken.clamp(0, N)
    base = taken.long() + need.cumsum(0) - need
    got = torch.minimum((N - base).clamp(min=0), need)
    add = torch.minimum(add, ((held + got) * BT - length).clamp(min=0))
    for r in range(len(length)):
        h, n, b = int(held[r]), int(got[r]), int(base[r])
        tables[r, h:h + n] = free[b:b + n]
    step = torch.arange(S, device=lengths.device)
    at = length[:, None] + step
    block = tables.long().gather(1, (at // BT).clamp(max=W - 1))
    there = (step < add[:, None]) & (block >= 0)
    return BlockPlan(torch.where(there, block * BT + at % BT, -1), torch.where(there, at, -1).int(), (length + add).int(),
                     (taken + got.sum()).int())


def _qkv_strides(qkv):
    """Strides of rows, tokens and groups of a packed projection that the kernels can read, or ``None``."""
    R, S, G, n, D = qkv.shape
    if qkv.stride(4) != 1 or qkv.stride(3) != D or qkv.data_ptr() % 16:
        return None
    strides = [0 if size == 1 else st for size, st in zip((R, S, G), qkv.stride())]
    return strides if all(st % 8 == 0 for st in strides) else None


def store_blocks(qkv, layer, slots, positions=None, rope_table=None) -> Optional[torch.Tensor]:
    """Store the keys and values of the packed projection output ``qkv [R, S, kv_heads, q_per_kv + 2, D]`` (per KV head: its query
    heads, then its key, then its value) at ``slots [R, S]`` of ``layer``, as ``plan_blocks`` gives them: the tokens of a row follow one
    another, those without a slot stand behind them (or in front, where the table lacks their block), and no block takes tokens of two rows.

    The scale of a block and head is the smallest power of two by which the largest finite value of its new tokens does not exceed the
    largest code (448 in e4m3, 127 in int8); a block that holds tokens already keeps the larger of its scale and that one, and where
    it grows its codes are rounded again.  Infinities become the largest code, NaN stays NaN in e4m3 and becomes 0 in int8.  Nothing
    behind the stored tokens is changed.

    With ``rope_table`` (``ops.rope_table``) and ``positions`` keys are stored rotated and the rotated queries are returned,
    ``[R, S, kv_heads * q_per_kv, D]`` (zeros for tokens without a slot); ``qkv`` is left as it is.  A token whose position the table
    lacks counts as one without a slot.  Without a table the result is ``None``."""
    if qkv.is_cuda and (host := host_paths()) is not None:
        out = host.store_blocks(qkv, *layer, slots, positions, rope_table)
        if out is not None:
            return out[0]
    dev = qkv.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return store_blocks(qkv, layer, slots, positions, rope_table)
    _check_layer(layer, 4)
    k, v, ks, vs = layer
    N, G, BT, D = k.shape
    if qkv.ndim != 5 or qkv.shape[2] != G or qkv.shape[3] < 2 or qkv.shape[4] != D:
        raise ValueError(f"qkv must be [R, S, {G}, q_per_kv + 2, {D}], not {list(qkv.shape)}")
    R, S, _, n, _ = qkv.shape
    if slots.dtype != torch.int64 or slots.shape != (R, S) or not slots.is_contiguous():
        raise ValueError(f"slots must be a dense int64 tensor of shape {[R, S]}, not {slots.dtype} {list(slots.shape)}")
    if rope_table is not None and positions is None:
        raise ValueError("a rope table needs the tokens' positions")
    if rope_table is not None:
        _int32("positions", positions, R, S)
        if rope_table.dtype != torch.float32 or rope_table.ndim != 3 or rope_table.shape[1:] != (D // 2, 2) or not rope_table.is_contiguous():
            raise ValueError(f"the rope table must be dense fp32 [positions, {D // 2}, 2]")
    _together(dev, qkv, k, v, ks, vs, slots, positions if rope_table is not None else None, rope_table)
    q = None if rope_table is None else torch.empty(R, S, G * (n - 2), D, dtype=qkv.dtype, device=dev)
    if R * S == 0 or N == 0 or G == 0:
        return q
    if not qkv.is_cuda:
        return _store_torch(qkv, layer, slots, positions, rope_table)
    if qkv.dtype not in _HALF:
        raise TypeError(f"store_blocks takes bf16 or fp16 on a GPU, not {qkv.dtype}")
    if D not in (64, 128):
        raise ValueError(f"store_blocks takes heads of 64 or 128 values on a GPU, not {D}")
    strides = _qkv_strides(qkv)
    if strides is None:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
        strides = _qkv_strides(qkv)
    if rope_table is not None and rope_table.data_ptr() % 16:
        rope_table = rope_table.clone()
    st = _lib.lib().axb_store_blocks(qkv.data_ptr(), *strides, slots.data_ptr(), _lib.addr(positions if rope_table is not None else None),
                                     _lib.addr(rope_table), _lib.addr(q), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), R, S,
                                     G, n - 2, D, N, BT, 0 if rope_table is None else rope_table.shape[0], _HALF[qkv.dtype],
                                     int(k.dtype == torch.int8), _lib.stream())
    _lib.check(st, "axb_store_blocks")
    return q


def _rotate_torch(x, table, positions):
    """``x [n, heads, D]`` at ``positions [n]``, fp32; every product is rounded by itself, as in the kernel."""
    h = x.shape[-1] // 2
    cs = table[positions.long()][:, None]
    a, b, cos, sin = x[..., :h], x[..., h:], cs[..., 0], cs[..., 1]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _scale_torch(largest, dtype):
    """The power of two for a largest magnitude."""
    top, most = (6, 127 / 64) if dtype == torch.int8 else (8, 448 / 256)
    m, e = torch.frexp(largest.double())                            # largest = 2 m 2^(e - 1)
    e = torch.where(largest > 0, e - 1 - top + (2 * m > most), LOWEST_EXPONENT).clamp(min=LOWEST_EXPONENT)
    return torch.exp2(e.double()).float()


def _codes_torch(x, dtype):
    if dtype == torch.int8:
        return x.nan_to_num(0.0, 127.0, -127.0).clamp(-127, 127).round().to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _store_torch(qkv, layer, slots, positions, table):
    k, v, ks, vs = layer
    N, G, BT, D = k.shape
    R, S, _, n, _ = qkv.shape
    slot = slots.reshape(-1)
    there = (slot >= 0) & (slot < N * BT)
    if table is not None:
        at = positions.reshape(-1)
        there &= (at >= 0) & (at < table.shape[0])
    slot, x = slot[there], qkv.detach().reshape(R * S, G, n, D)[there].float()
    q = None
    if table is not None:
        turned = _rotate_torch(x[:, :, :-1].reshape(len(x), G * (n - 1), D), table, at[there]).view(len(x), G, n - 1, D)
        q = torch.zeros(R * S, G, n - 2, D, dtype=qkv.dtype, device=qkv.device)
        q[there] = turned[:, :, :-1].to(qkv.dtype)
        q = q.view(R, S, G * (n - 2), D)
        x = torch.cat([turned, x[:, :, -1:]], 2)
    block, place = slot // BT, slot % BT
    for codes, scales, y in ((k, ks, x[:, :, -2]), (v, vs, x[:, :, -1])):
        raw = codes.view(torch.uint8)
        for b in block.unique().tolist():
            mine = block == b
            held = int(place[mine].min())
            size = y[mine].abs()
            scale = _scale_torch(torch.where(size <= torch.finfo(torch.float32).max, size, 0).amax((0, 2)), codes.dtype)
            if held:
                scale = torch.maximum(scale, scales[b])
                shrink = (scales[b] / scale)[:, None, None]
                old = codes[b, :, :held].float()
                raw[b, :, :held] = torch.where(shrink < 1, _codes_torch(old * shrink, codes.dtype).view(torch.uint8), raw[b, :, :held])
            scales[b] = scale
            raw[b, :, place[mine]] = _codes_torch(y[mine] / scale[:, None], codes.dtype).view(torch.uint8).transpose(0, 1)
    return q


def cached_attention(q, layer, tables, lengths, new=None, scale=None):
    """Attention of new tokens over the cache, which holds their own keys and values already: ``q [R, S, heads, D]`` (or
    ``[R, S, kv_heads, q_per_kv, D]``, such as the query part of a packed projection output) against the ``lengths[r]`` tokens that the
    blocks of ``tables[r]`` hold.  The first ``new[r]`` queries of a row (``None``: all S) are the last tokens of the sequence, and each
    sees the tokens up to its own; the queries behind them, and those of an empty sequence, give zeros.  Returns
    ``[R, S, heads, D]`` in the type of ``q``.

    Blocks that a table lacks (-1 within the length) count as absent.  What lies behind a sequence in its last block is never
    looked at.  On a GPU: bf16 or fp16, D 64 or 128; scores, sums and denominators are 32-bit, and softmax weights are rounded to fp16 (half
    a step, 2^-11, of each down to e^-18 of a query's largest one, smaller ones by less than 2^-37 of that); the work is bound by reading the cache, once for up to 16 query columns
    (``S * q_per_kv``); more than 48 share the reading in groups of 128 on the tensor cores' own memory.  A prompt that starts a
    sequence is better evaluated with ``flash_attention`` before it is stored."""
    if q.is_cuda and (host := host_paths()) is not None:
        out = host.cached_attention(q, *layer, tables, lengths, new, scale)
        if out is not None:
            return out
    dev = q.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return cached_attention(q, layer, tables, lengths, new, scale)
    _check_layer(layer, 4)
    k, v, ks, vs = layer
    N, G, BT, D = k.shape
    shape = q.shape
    if q.ndim == 4 and G and shape[2] % G == 0 and shape[3] == D:
        R, S, H, _ = shape
        strides, head = (q.stride(0), q.stride(1), H // G * q.stride(2)), q.stride(2)
    elif q.ndim == 5 and shape[2] == G and shape[4] == D:
        R, S, H = shape[0], shape[1], G * shape[3]
        strides, head = q.stride()[:3], q.stride(3)
    else:
        raise ValueError(f"q must be [R, S, heads, {D}] with a multiple of {G} heads, or [R, S, {G}, q_per_kv, {D}], not {list(shape)}")
    if tables.ndim != 2:
        raise ValueError("tables must be [R, W]")
    _int32("tables", tables, R, tables.shape[1])
    _int32("lengths", lengths, R)
    if new is not None:
        _int32("new", new, R)
    _together(dev, q, k, v, ks, vs, tables, lengths, new)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if not math.isfinite(scale):
        raise ValueError("the softmax scale must be finite")
    P = H // G if G else 0
    if R * S * H == 0 or N == 0 or tables.shape[1] == 0:
        return torch.zeros(R, S, H, D, dtype=q.dtype, device=dev)
    if not q.is_cuda:
        return _attend_torch(q.reshape(R, S, G, P, D), layer, tables, lengths, new, scale)
    if q.dtype not in _HALF:
        raise TypeError(f"cached_attention takes bf16 or fp16 on a GPU, not {q.dtype}")
    if D not in (64, 128):
        raise ValueError(f"cached_attention takes heads of 64 or 128 values on a GPU, not {D}")
    strides = [0 if size == 1 else st for size, st in zip((R, S, G), strides)]
    if q.stride(-1) != 1 or (head != D and P > 1) or any(st % 8 for st in strides) or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        strides = (S * H * D, H * D, P * D)
    out = torch.empty(R, S, H, D, dtype=q.dtype, device=dev)
    L = _lib.lib()
    work = torch.empty(L.axb_cached_attention_words(R, S, G, P, D), dtype=torch.float32, device=dev)
    st = L.axb_cached_attention(q.data_ptr(), *strides, k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), tables.data_ptr(),
                                lengths.data_ptr(), _lib.addr(new), out.data_ptr(), work.data_ptr(), R, S, G, P, D, tables.shape[1], N,
                                BT, scale, _HALF[q.dtype], int(k.dtype == torch.int8), _lib.stream())
    _lib.check(st, "axb_cached_attention")
    _lib.add_launches(1)
    return out


def _attend_torch(q, layer, tables, lengths, new, scale):
    R, S, G, P, D = q.shape
    N, _, BT, _ = layer.k.shape
    out = torch.zeros(R, S, G, P, D, dtype=q.dtype, device=q.device)
    for r in range(R):
        n = min(max(int(lengths[r]), 0), tables.shape[1] * BT)
        m = S if new is None else min(max(int(new[r]), 0), S)
        if n == 0 or m == 0:
            continue
        ids = tables[r, :(n + BT - 1) // BT].long()
        there = ((ids >= 0) & (ids < N)).repeat_interleave(BT)[:n]
        ids = ids.clamp(0, N - 1)
        k, v = ((c[ids].float() * s[ids][..., None, None]).transpose(1, 2).reshape(-1, G, D)[:n]
                for c, s in ((layer.k, layer.k_scale), (layer.v, layer.v_scale)))
        at = n - m + torch.arange(m, device=q.device)               # the token that a query stands at
        seen = there & (torch.arange(n, device=q.device) <= at[:, None])
        a = torch.einsum("sgpd,tgd->gpst", q[r, :m].float(), k) * scale
        a = a.masked_fill(~seen, float("-inf"))
        p = (a - a.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp().masked_fill(~seen, 0)
        total = p.sum(-1, keepdim=True)
        for s in range(m):                                          # what a query does not see may be NaN
            vis = seen[s]
            if bool(vis.any()):
                out[r, s] = (torch.einsum("gpt,tgd->gpd", p[:, :, s, vis], v[vis]) / total[:, :, s]).to(q.dtype)
    return out.view(R, S, G * P, D)


def reorder_blocks(blocks, tables, lengths, spare, parents):
    """Rows go on from other rows, as the beams of a prompt do: row ``j`` of group ``b`` from row ``parents[b, j]`` of that group.

    ``blocks``: a ``BlockLayer`` of all layers, stacked in front (``[layers, blocks, kv_heads, block_tokens, D]``); ``tables [R, W]``,
    ``lengths [R]`` with ``R = groups * beams`` rows, those of a group equally long, ``parents [groups, beams]`` (int32).  Full blocks are shared by naming them.  The
    block that a row still writes into is its own: a row with another parent has its parent's unfinished block copied into the block
    ``spare[r]``, and keeps the block that it leaves as the new spare one; ``spare [R]`` and the unfinished blocks of the rows are all
    different.  Returns the rows' new ``(tables, lengths, spare)``; the arguments are left as they are, but for the contents of the
    spare blocks.  A parent outside the group counts as the row itself."""
    if tables.is_cuda and (host := host_paths()) is not None:
        out = host.reorder_blocks(*blocks, tables, lengths, spare, parents)
        if out is not None:
            return out
    dev = tables.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return reorder_blocks(blocks, tables, lengths, spare, parents)
    _check_layer(blocks, 5)
    if tables.ndim != 2 or parents.ndim != 2:
        raise ValueError("reorder_blocks takes tables [R, W] and parents [groups, beams]")
    R, W = tables.shape
    _int32("tables", tables, R, W)
    _int32("lengths", lengths, R)
    _int32("spare", spare, R)
    _int32("parents", parents, *parents.shape)
    if parents.numel() != R:
        raise ValueError(f"{list(parents.shape)} parents for {R} rows")
    _together(dev, *blocks, lengths, spare, parents)
    k, v, ks, vs = blocks
    layers, N, G, BT, D = k.shape
    if R == 0 or W == 0 or k.numel() == 0:
        return tables.clone(), lengths.clone(), spare.clone()
    if not tables.is_cuda:
        return _reorder_torch(blocks, tables, lengths, spare, parents)
    if D % 16:
        raise ValueError(f"reorder_blocks takes heads of a multiple of 16 values on a GPU, not {D}")
    out = torch.empty_like(tables), torch.empty_like(lengths), torch.empty_like(spare)
    st = _lib.lib().axb_reorder_blocks(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), tables.data_ptr(), lengths.data_ptr(),
                                       spare.data_ptr(), parents.data_ptr(), *(t.data_ptr() for t in out), layers, R, parents.shape[1], W,
                                       N, G, BT, D, _lib.stream())
    _lib.check(st, "axb_reorder_blocks")
    return out


def _reorder_torch(blocks, tables, lengths, spare, parents):
    K, BT, N = parents.shape[1], blocks.k.shape[3], blocks.k.shape[1]
    row = torch.arange(tables.shape[0])
    parent = parents.reshape(-1).long()
    parent = row // K * K + torch.where((parent >= 0) & (parent < K), parent, row % K)
    new_tables, new_lengths, new_spare = tables[parent], lengths[parent], spare.clone()
    for r, p in enumerate(parent.tolist()):
        full, part = divmod(max(int(lengths[p]), 0), BT)
        if p == r or part == 0 or full >= tables.shape[1]:
            continue
        source, target = int(tables[p, full]), int(spare[r])
        new_tables[r, full], new_spare[r] = spare[r], tables[r, full]
        if 0 <= source < N and 0 <= target < N:
            for c in blocks[:2]:
                c.view(torch.uint8)[:, target, :, :part] = c.view(torch.uint8)[:, source, :, :part]
            for s in blocks[2:]:
                s[:, target] = s[:, source]
    return new_tables, new_lengths, new_spare
