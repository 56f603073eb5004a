"""Greedy decoding and beam search with the tensor-parallel language models (inference through the same layers and kernels).

The reference runs inference by handing its patched Hugging Face models to ``generate``; the models of this
package return logits whose vocabulary dimension is split over the ranks of ``model.head.group``, so choosing the
next token is a small collective: every rank proposes its best local candidate and all ranks pick the same winner.
"""

import torch
import torch.distributed as dist

from .. import ops
from ..intra_layer.communication import _gather
from .cache import BlockCache


@torch.no_grad()
def parallel_argmax(logits, group=None):
    """``argmax`` over a last dimension that is split over ``group`` in rank order (``None``: not split).  Every
    rank returns the same global indices; ties go to the lowest index, as in ``torch.argmax`` of the whole row."""
    value, index = logits.float().max(dim=-1)
    if group is None or dist.get_world_size(group) == 1:
        return index
    n, me = dist.get_world_size(group), dist.get_rank(group)
    index = index + me * logits.shape[-1]
    values = [torch.empty_like(value) for _ in range(n)]
    indices = [torch.empty_like(index) for _ in range(n)]
    dist.all_gather(values, value.contiguous(), group=group)
    dist.all_gather(indices, index.contiguous(), group=group)
    values, indices = torch.stack(values, -1), torch.stack(indices, -1)      # [..., n]; rank order = index order
    best = values.argmax(dim=-1, keepdim=True)                               # first maximum = lowest rank
    return indices.gather(-1, best).squeeze(-1)


@torch.no_grad()
def greedy_generate(model, tokens, max_new_tokens: int, eos_id=None, cache_dtype=None, prompt_lengths=None, block_tokens=64):
    """Extend ``tokens`` ``[B, S0]`` by up to ``max_new_tokens`` greedily chosen tokens; returns ``[B, S0 + new]``.

    Every rank of a tensor-parallel group passes the same ``tokens`` (ranks that differ in data or depth
    coordinates may pass different batches).  Without ``cache_dtype`` the whole prefix is re-evaluated for every new token (no
    key/value cache), which keeps the attention kernels' training-time code path; sequences stop growing for rows that have
    produced ``eos_id``, which are padded with it.  The model is left in evaluation mode for the call.

    With ``cache_dtype`` (``torch.float8_e4m3fn`` or ``torch.int8``) keys and values are kept in a ``BlockCache`` with blocks of
    ``block_tokens`` and every token is evaluated once; scores differ by the rounding of what is stored.  Prompts may then differ in
    length: row ``r`` is ``tokens[r, :prompt_lengths[r]]``, and its new tokens follow there; what is left of a row is ``eos_id`` (or 0).
    A ``Mixtral``'s expert capacity is that of a step's tokens, one per row, padding of the prompts among them: what is dropped differs
    from an evaluation of whole prefixes unless ``capacity_factor`` leaves room for all."""
    if cache_dtype is None and prompt_lengths is not None:
        raise ValueError("prompts of different lengths need a cache (cache_dtype)")
    was_training = model.training
    model.eval()
    limit = getattr(getattr(model, "cfg", None), "seq_len", None)
    if cache_dtype is not None:
        try:
            return _greedy_cached(model, tokens, max_new_tokens, eos_id, limit, cache_dtype, prompt_lengths, block_tokens)
        finally:
            model.train(was_training)
    done = torch.zeros(tokens.shape[0], dtype=torch.bool, device=tokens.device)
    try:
        for _ in range(max_new_tokens):
            if limit is not None and tokens.shape[1] >= limit:
                break
            logits = model(tokens)                                           # [B, S, vocab / |group|]
            nxt = parallel_argmax(logits[:, -1], getattr(model.head, "group", None)).to(tokens.dtype)
            if eos_id is not None:
                nxt = torch.where(done, torch.full_like(nxt, eos_id), nxt)
                done = done | (nxt == eos_id)
            tokens = torch.cat([tokens, nxt[:, None]], dim=1)
            if eos_id is not None and bool(done.all()):
                break
    finally:
        model.train(was_training)
    return tokens


def _prompt(tokens, max_new_tokens, limit, prompt_lengths):
    """(lengths int32 on the device, longest of them, number of new tokens that the model's length leaves)."""
    B, S = tokens.shape
    if B == 0 or S == 0:
        raise ValueError("generation with a cache starts from a prompt")
    if limit is not None and S > limit:
        raise ValueError(f"prompts of {S} tokens, of which the model takes {limit}")
    if prompt_lengths is None:
        lengths = torch.full((B,), S, dtype=torch.int32, device=tokens.device)
    else:
        lengths = torch.as_tensor(prompt_lengths, device=tokens.device).to(torch.int32)
        if lengths.shape != (B,) or int(lengths.min()) < 1 or int(lengths.max()) > S:
            raise ValueError(f"prompt_lengths must be {B} numbers from 1 to {S}")
    room = max_new_tokens if limit is None else min(max_new_tokens, limit - S)
    return lengths, max(room, 0)


def _greedy_cached(model, tokens, max_new_tokens, eos_id, limit, dtype, prompt_lengths, block_tokens):
    lengths, room = _prompt(tokens, max_new_tokens, limit, prompt_lengths)
    B, S = tokens.shape
    pad = 0 if eos_id is None else eos_id
    out = torch.full((B, S + room), pad, dtype=tokens.dtype, device=tokens.device)
    out[:, :S] = torch.where(torch.arange(S, device=tokens.device) < lengths[:, None], tokens, pad)
    if room == 0:
        return out
    cache = BlockCache(model, B, S + room, block_tokens, dtype)
    done = torch.zeros(B, dtype=torch.bool, device=tokens.device)
    cache.plan(S, lengths)
    step, at = tokens, lengths.long()[:, None]
    for i in range(room):
        logits = model(step, cache=cache)                                    # [B, 1, vocab / |group|]
        nxt = parallel_argmax(logits[:, -1], getattr(model.head, "group", None)).to(tokens.dtype)
        if eos_id is not None:
            nxt = torch.where(done, torch.full_like(nxt, eos_id), nxt)
            done = done | (nxt == eos_id)
        step = nxt[:, None]
        out.scatter_(1, at + i, step)
        if eos_id is not None and bool(done.all()):
            return out[:, :S + i + 1]
        if i + 1 < room:
            cache.plan(1)
    return out


@torch.no_grad()
def beam_generate(model, tokens, max_new_tokens: int, beams: int, eos_id=None, length_penalty: float = 0.0, cache_dtype=torch.float8_e4m3fn,
                  prompt_lengths=None, block_tokens=64):
    """Beam search: the ``beams`` (up to 32) continuations of every prompt of ``tokens`` ``[B, S0]`` with the largest sums of
    log-probabilities that are found.  Returns ``(sequences [B, beams, S0 + new], scores [B, beams])``, best first.

    A beam ends with ``eos_id`` and is padded with it, its score then stands; at the end scores are divided by the number of new
    tokens (the end token included) to the power of ``length_penalty``.  Prompts are evaluated once, into a ``BlockCache`` whose full
    blocks the beams share.  ``cache_dtype``, ``prompt_lengths`` and ``block_tokens`` as for ``greedy_generate``; every rank of a
    tensor-parallel group passes the same ``tokens`` and gets the same result.  The model is left in evaluation mode for the call."""
    was_training = model.training
    model.eval()
    limit = getattr(getattr(model, "cfg", None), "seq_len", None)
    try:
        lengths, room = _prompt(tokens, max_new_tokens, limit, prompt_lengths)
        B, S = tokens.shape
        device, group = tokens.device, getattr(model.head, "group", None)
        if not 1 <= beams <= ops.MOST_BEAMS:
            raise ValueError(f"1 to {ops.MOST_BEAMS} beams, not {beams}")
        pad = 0 if eos_id is None else eos_id
        out = torch.full((B, beams, S + room), pad, dtype=tokens.dtype, device=device)
        out[:, :, :S] = torch.where(torch.arange(S, device=device) < lengths[:, None], tokens, pad)[:, None]
        scores = torch.full((B, beams), float("-inf"), device=device)
        scores[:, 0] = 0.0
        if room == 0:
            return out, scores
        cache = BlockCache(model, B, S + room, block_tokens, cache_dtype, beams, S)
        done = None if eos_id is None else torch.zeros(B, beams, dtype=torch.bool, device=device)
        count = torch.zeros(B, beams, dtype=torch.int64, device=device)      # new tokens of every beam
        cache.plan(S, lengths)
        step, at, length = tokens, lengths.long()[:, None, None].expand(B, beams, 1), S
        for i in range(room):
            logits = model(step, cache=cache)[:, -1]
            if group is not None:
                logits = _gather(logits, -1, group)
            if i == 0:                                                       # all beams start from the prompt
                logits = logits[:, None].expand(-1, beams, -1)
                cache.expand(beams)
            best = ops.beam_select(logits.reshape(B, beams, -1), scores, done, eos_id)
            parents = best.parents.long()
            if done is not None:
                count = torch.where(done.gather(1, parents), count.gather(1, parents), i + 1)
            out = out.gather(1, parents[..., None].expand_as(out)).scatter_(2, at + i, best.tokens[..., None].to(tokens.dtype))
            scores, done, length = best.scores, best.done, S + i + 1
            if done is not None and bool(done.all()):
                break
            if i + 1 < room:
                cache.reorder(best.parents)
                cache.plan(1)
                step = best.tokens.view(B * beams, 1)
        if done is None:
            count = torch.full_like(count, room)
        scores = scores / count.clamp(min=1).to(scores.dtype) ** length_penalty
        scores, order = scores.sort(dim=1, descending=True, stable=True)
        return out.gather(1, order[..., None].expand_as(out))[:, :, :length], scores
    finally:
        model.train(was_training)
