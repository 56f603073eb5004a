"""Rows of a table by token, scaled, with the gradient by sorted tokens (``csrc/embedding.cu``)."""

import math

import torch
import torch.nn.functional as F

from . import _lib
from .direct import batched, host_paths, no_graph, plain_tensors
from .gemm import as_written
from .kv_cache import _elsewhere

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_INDEX = {torch.int32: 4, torch.int64: 8}
EMBEDDING_TYPES = tuple(_DT)


def embedding(tokens, weight, scale=1.0, padding_idx=None):
    """``weight[tokens] * scale``: ``tokens [...]`` (int32 or int64), ``weight [V, H]`` (bf16, fp16 or fp32), returns ``[..., H]`` in the type
    of ``weight``, each value rounded once (magnitudes below 2^-126 are kept).

    The gradient of ``weight`` has the sums of the rows of equal tokens, 32-bit in an order that the tokens alone decide (the same bits on
    every run), scaled and rounded once; ``padding_idx`` gets none.  Gradients of gradients are lookups again.  A token outside the table
    gives a row of NaN and no gradient on a GPU, and is an error on the CPU.  The call never synchronises and can be captured into a CUDA graph."""
    if weight.is_cuda and (host := host_paths()) is not None:
        out = host.embedding(tokens, weight, scale, -1 if padding_idx is None else padding_idx if padding_idx >= 0 else -2)
        if out is not None:
            return out
    if weight.ndim != 2 or weight.dtype not in _DT:
        raise ValueError(f"weight must be [V, H] in bf16, fp16 or fp32, not {weight.dtype} {list(weight.shape)}")
    if tokens.dtype not in _INDEX:
        raise ValueError(f"tokens must be int32 or int64, not {tokens.dtype}")
    if tokens.device != weight.device:
        raise ValueError(f"tensors on {weight.device} and {tokens.device}")
    if not math.isfinite(scale):
        raise ValueError(f"the scale is a finite number, not {scale}")
    V = weight.shape[0]
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {V} rows")
        if padding_idx < 0:
            return embedding(tokens, weight, scale, padding_idx + V)
    if not plain_tensors(tokens, weight) or weight.numel() == 0 or V > 1 << 30 or weight.shape[1] > 1 << 25 or tokens.numel() >= 1 << 31:
        return _torch(tokens, weight, scale, padding_idx)
    if _elsewhere(weight.device):
        with torch.cuda.device(weight.device):
            return embedding(tokens, weight, scale, padding_idx)
    if no_graph(weight):
        return _rows(tokens, weight, scale)[0]
    return _EmbeddingFn.apply(tokens, weight, scale, -1 if padding_idx is None else padding_idx)


def _torch(tokens, weight, scale, padding_idx):
    out = F.embedding(tokens, weight, padding_idx)
    return out if scale == 1.0 else (out.float() * scale).to(weight.dtype)


def _rows(tokens, weight, scale, padding=-1, sort=False):
    """``weight[tokens] * scale``; with ``sort`` also what the gradient needs of the tokens."""
    weight = weight.detach()
    if weight.shape[1] > 1 and weight.stride(1) != 1:
        weight = weight.contiguous()
    tokens, (V, H), L = tokens.contiguous(), weight.shape, _lib.lib()
    out = torch.empty(*tokens.shape, H, dtype=weight.dtype, device=weight.device)
    sorted_ = torch.empty(L.axb_embedding_sorted_words(tokens.numel(), V), dtype=torch.int32, device=weight.device) if sort else None
    if out.numel():
        st = L.axb_embedding(tokens.data_ptr(), _INDEX[tokens.dtype], tokens.numel(), weight.data_ptr(), weight.stride(0), V, H, scale, out.data_ptr(),
                             padding, _lib.addr(sorted_), _DT[weight.dtype], _lib.stream())
        _lib.check(st, "axb_embedding")
        _lib.add_launches(int(sort and sorted_.numel() > 0))
    return out, sorted_


def _table_gradient(tokens, sorted_, dy, V, scale, padding):
    """``dy [..., H]`` summed by token; the rows may have any stride."""
    H = dy.shape[-1]
    dy = dy.reshape(-1, H)
    if H > 1 and dy.stride(1) != 1:
        dy = dy.contiguous()
    n, L, tokens = dy.shape[0], _lib.lib(), tokens.contiguous()
    out = torch.empty(V, H, dtype=dy.dtype, device=dy.device)
    work = torch.empty(L.axb_embedding_grad_words(n, H), dtype=torch.int32, device=dy.device)
    st = L.axb_embedding_grad(tokens.data_ptr(), _INDEX[tokens.dtype], sorted_.data_ptr(), n, dy.data_ptr(), dy.stride(0), V, H, scale, padding,
                              out.data_ptr(), work.data_ptr(), _DT[dy.dtype], _lib.stream())
    _lib.check(st, "axb_embedding_grad")
    _lib.add_launches(-1 if n == 0 else int(sorted_.numel() > 0))
    return out


def _batched_gradient(tokens, dy, V, scale, padding):
    """Of a gradient that stands for many (``is_grads_batched``, vectorised Jacobians): a wrapper without memory of its own, which torch's
    operators know.  Sums in 32 bits; tokens without a gradient go to a row behind the table's."""
    none = (tokens < 0) | (tokens >= V) | (tokens == padding)
    sums = torch.ops.aten.embedding_dense_backward(dy.float(), tokens.long().masked_fill(none, V), V + 1, -1, False)
    return (sums[:V] * scale).to(dy.dtype)


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        out, sorted_ = _rows(tokens, weight, scale, padding, True)
        ctx.save_for_backward(tokens, sorted_)
        ctx.scale, ctx.padding, ctx.V = scale, padding, weight.shape[0]
        return out

    @staticmethod
    def backward(ctx, dy):
        if batched(dy) or not plain_tensors(dy):
            return None, _batched_gradient(ctx.saved_tensors[0], dy, ctx.V, ctx.scale, ctx.padding), None, None
        return None, _EmbeddingGradFn.apply(*ctx.saved_tensors, dy, ctx.V, ctx.scale, ctx.padding), None, None


class _EmbeddingGradFn(torch.autograd.Function):
    """The gradient of the table as a function of that of the rows, and its own: rows of the table that it is asked with."""

    @staticmethod
    def forward(ctx, tokens, sorted_, dy, V, scale, padding):
        ctx.save_for_backward(tokens)
        ctx.scale, ctx.padding = scale, padding
        return _table_gradient(tokens, as_written(sorted_), dy, V, scale, padding)

    @staticmethod
    def backward(ctx, d_table):
        (tokens,) = ctx.saved_tensors
        V = d_table.shape[0]
        none = (tokens < 0) | (tokens >= V) | (tokens == ctx.padding)
        rows = embedding(tokens.masked_fill(none, 0), d_table, ctx.scale)
        return None, None, rows.masked_fill(none[..., None], 0), None, None, None
