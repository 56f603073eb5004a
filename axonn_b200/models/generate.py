"""Greedy decoding, beam search and scoring with the tensor-parallel language models (inference through the same layers and kernels).

The reference runs inference by handing its patched Hugging Face models to ``generate``; the models of this
package return logits whose vocabulary dimension is split over the ranks of ``model.head.group``, so choosing the
next token is a small collective: every rank proposes its best local candidate and all ranks pick the same winner.
"""

import torch
import torch.distributed as dist

from .. import ops
from ..intra_layer.communication import _gather
from .cache import BlockCache

_LEFT_OUT = -100


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


def _of_the_table(model, tokens, there):
    """``tokens`` with a token of the model's vocabulary wherever they are not ``there`` and none (-1, a label's -100): of such a number a GPU's
    lookup makes NaN, which attention hands on to the tokens in front of it (a weight of zero times NaN)."""
    vocab = getattr(getattr(model, "cfg", None), "vocab", None)
    return tokens if vocab is None else torch.where(there | (tokens >= 0) & (tokens < vocab), tokens, 0)


def score_tokens(model, tokens, lengths=None, entropy=False, top=0, temperature=1.0):
    """What ``model`` makes of given sequences: the ``ops.TokenLogProbs`` of ``tokens[:, 1:]`` (``tokens [B, S]``, int64), each after the
    tokens in front of it, all of shape ``[B, S - 1]``.  Row ``r`` is ``tokens[r, :lengths[r]]`` (``None``: all of it); behind that any
    numbers may stand, and the results are zeros (alternatives -1).  With gradients enabled the results are functions of the model's
    parameters: a policy-gradient or distillation loss is a sum of them.  Every rank of a tensor-parallel group passes the same ``tokens``."""
    if tokens.ndim != 2 or tokens.dtype != torch.int64 or tokens.shape[1] < 2:
        raise ValueError(f"sequences of two tokens and more are scored, int64 [B, S], not {tokens.dtype} {list(tokens.shape)}")
    if hasattr(model, "pos_emb") and tokens.shape[1] > model.cfg.seq_len:
        raise ValueError(f"sequences of {tokens.shape[1]} tokens for a model that has learned {model.cfg.seq_len} positions")
    targets = tokens[:, 1:]
    if lengths is not None:
        lengths = torch.as_tensor(lengths, device=tokens.device)
        if lengths.shape != tokens.shape[:1]:
            raise ValueError(f"lengths must be {tokens.shape[0]} numbers, not {list(lengths.shape)}")
        there = torch.arange(tokens.shape[1], device=tokens.device) < lengths[:, None]
        targets = targets.masked_fill(~there[:, 1:], _LEFT_OUT)
        tokens = _of_the_table(model, tokens, there)
    logits = model(tokens)                                                   # [B, S, vocab / |group|]
    return ops.token_log_probs(logits[:, :-1], targets, entropy, top, temperature, getattr(model.head, "group", None), _LEFT_OUT)


class _Told:
    """Log-probabilities of the new tokens of a batch, step by step, with ``top`` alternatives."""

    def __init__(self, top, group):
        self.top, self.group, self.steps = top, group, []

    def step(self, logits, tokens, done):
        if done is not None:
            tokens = tokens.masked_fill(done, _LEFT_OUT)
        self.steps.append(ops.token_log_probs(logits, tokens, top=self.top, group=self.group, ignore_index=_LEFT_OUT))

    def result(self, rows, device):
        if self.steps:
            return ops.TokenLogProbs(*(None if t[0] is None else torch.stack(t, 1) for t in zip(*self.steps)))
        none = torch.empty(rows, 0, device=device)
        best = none.new_empty(rows, 0, self.top) if self.top else None
        return ops.TokenLogProbs(none, None, best, None if best is None else best.long())


@torch.no_grad()
def greedy_generate(model, tokens, max_new_tokens: int, eos_id=None, cache_dtype=None, prompt_lengths=None, block_tokens=64, alternatives=None):
    """Extend ``tokens`` ``[B, S0]`` by up to ``max_new_tokens`` greedily chosen tokens; returns ``[B, S0 + new]``.

    Every rank of a tensor-parallel group passes the same ``tokens`` (ranks that differ in data or depth
    coordinates may pass different batches).  Without ``cache_dtype`` the whole prefix is re-evaluated for every new token (no
    key/value cache), which keeps the attention kernels' training-time code path; sequences stop growing for rows that have
    produced ``eos_id``, which are padded with it.  The model is left in evaluation mode for the call.

    With ``cache_dtype`` (``torch.float8_e4m3fn`` or ``torch.int8``) keys and values are kept in a ``BlockCache`` with blocks of
    ``block_tokens`` and every token is evaluated once; scores differ by the rounding of what is stored.  Prompts may then differ in
    length: row ``r`` is ``tokens[r, :prompt_lengths[r]]`` (behind that any numbers may stand), and its new tokens follow there; what is left of a
    row is ``eos_id`` (or 0).
    A ``Mixtral``'s expert capacity is that of a step's tokens, one per row, padding of the prompts among them: what is dropped differs
    from an evaluation of whole prefixes unless ``capacity_factor`` leaves room for all.

    With ``alternatives`` (0 to 32) the result is ``(tokens, ops.TokenLogProbs)``: the log-probabilities ``[B, new]`` of the new tokens,
    and as many of the likeliest tokens at each of their places; zeros (-1) for rows that have ended."""
    if cache_dtype is None and prompt_lengths is not None:
        raise ValueError("prompts of different lengths need a cache (cache_dtype)")
    if alternatives is not None and not 0 <= alternatives <= ops.MOST_ALTERNATIVES:
        raise ValueError(f"0 to {ops.MOST_ALTERNATIVES} alternatives, not {alternatives}")
    told = None if alternatives is None else _Told(alternatives, getattr(model.head, "group", None))
    was_training = model.training
    model.eval()
    limit = getattr(getattr(model, "cfg", None), "seq_len", None)
    if cache_dtype is not None:
        try:
            out = _greedy_cached(model, tokens, max_new_tokens, eos_id, limit, cache_dtype, prompt_lengths, block_tokens, told)
        finally:
            model.train(was_training)
        return out if told is None else (out, told.result(tokens.shape[0], tokens.device))
    done = torch.zeros(tokens.shape[0], dtype=torch.bool, device=tokens.device)
    try:
        for _ in range(max_new_tokens):
            if limit is not None and tokens.shape[1] >= limit:
                break
            logits = model(tokens)                                           # [B, S, vocab / |group|]
            nxt = parallel_argmax(logits[:, -1], getattr(model.head, "group", None)).to(tokens.dtype)
            if told is not None:
                told.step(logits[:, -1], nxt.long(), done if eos_id is not None else None)
            if eos_id is not None:
                nxt = torch.where(done, torch.full_like(nxt, eos_id), nxt)
                done = done | (nxt == eos_id)
            tokens = torch.cat([tokens, nxt[:, None]], dim=1)
            if eos_id is not None and bool(done.all()):
                break
    finally:
        model.train(was_training)
    return tokens if told is None else (tokens, told.result(tokens.shape[0], tokens.device))


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


def _greedy_cached(model, tokens, max_new_tokens, eos_id, limit, dtype, prompt_lengths, block_tokens, told):
    lengths, room = _prompt(tokens, max_new_tokens, limit, prompt_lengths)
    B, S = tokens.shape
    pad = 0 if eos_id is None else eos_id
    out = torch.full((B, S + room), pad, dtype=tokens.dtype, device=tokens.device)
    there = torch.arange(S, device=tokens.device) < lengths[:, None]
    out[:, :S] = torch.where(there, tokens, pad)
    if room == 0:
        return out
    cache = BlockCache(model, B, S + room, block_tokens, dtype)
    done = torch.zeros(B, dtype=torch.bool, device=tokens.device)
    cache.plan(S, lengths)
    step, at = tokens if prompt_lengths is None else _of_the_table(model, tokens, there), lengths.long()[:, None]
    for i in range(room):
        logits = model(step, cache=cache)                                    # [B, 1, vocab / |group|]
        nxt = parallel_argmax(logits[:, -1], getattr(model.head, "group", None)).to(tokens.dtype)
        if told is not None:
            told.step(logits[:, -1], nxt.long(), done if eos_id is not None else None)
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
        there = torch.arange(S, device=device) < lengths[:, None]
        out[:, :, :S] = torch.where(there, tokens, pad)[:, None]
        scores = torch.full((B, beams), float("-inf"), device=device)
        scores[:, 0] = 0.0
        if room == 0:
            return out, scores
        cache = BlockCache(model, B, S + room, block_tokens, cache_dtype, beams, S)
        done = None if eos_id is None else torch.zeros(B, beams, dtype=torch.bool, device=device)
        count = torch.zeros(B, beams, dtype=torch.int64, device=device)      # new tokens of every beam
        cache.plan(S, lengths)
        step = tokens if prompt_lengths is None else _of_the_table(model, tokens, there)
        at, length = lengths.long()[:, None, None].expand(B, beams, 1), S
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
