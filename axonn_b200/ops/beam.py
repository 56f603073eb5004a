"""Selection of beam search (``csrc/beam.cu``)."""

from typing import NamedTuple, Optional

import torch

from . import _lib
from .direct import host_paths
from .kv_cache import _elsewhere, _together

MOST_BEAMS = 32
_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class BeamStep(NamedTuple):
    """The best continuations of every prompt, best first: ``scores``, ``tokens`` (int64), ``parents`` (int32, the beam that each goes on
    from) and ``done`` (bool, or ``None``), all ``[prompts, beams]``."""

    scores: torch.Tensor
    tokens: torch.Tensor
    parents: torch.Tensor
    done: Optional[torch.Tensor]


def beam_select(logits, scores, done=None, eos_id=None):
    """The ``beams`` best of all continuations of a prompt's beams: ``logits [prompts, beams, vocabulary]``, ``scores [prompts, beams]``
    (fp32, sums of log-probabilities; ``-inf``: nothing goes on from that beam, as from all but the first at the start).

    A continuation's value is the beam's score plus the log-probability of the token; equal values count in the order of (beam, token),
    and a beam's tokens in the order of their logits.  Of a beam that is ``done`` (bool) only ``eos_id`` goes on, at the beam's score;
    the two are given together.  A value that is not a number counts as ``-inf``, and so do a score of ``+inf`` and all of a beam
    whose logits sum up to none (a NaN or ``+inf`` among them, or all ``-inf``).  Up to 32 beams.

    On a GPU a beam's sum is exact to 2^-18: candidates of two beams whose values are closer may change places."""
    if logits.is_cuda and (host := host_paths()) is not None:
        out = host.beam_select(logits, scores, done, eos_id)
        if out is not None:
            return BeamStep(*out)
    dev = logits.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return beam_select(logits, scores, done, eos_id)
    if logits.ndim != 3 or logits.dtype not in _DT or logits.shape[2] == 0:
        raise ValueError(f"logits must be [prompts, beams, vocabulary] in bf16, fp16 or fp32, not {logits.dtype} {list(logits.shape)}")
    B, K, V = logits.shape
    if not 1 <= K <= MOST_BEAMS:
        raise ValueError(f"1 to {MOST_BEAMS} beams, not {K}")
    if V > 1 << 30:
        raise ValueError(f"a vocabulary of at most {1 << 30}, not {V}")
    if scores.dtype != torch.float32 or scores.shape != (B, K):
        raise ValueError(f"scores must be fp32 {[B, K]}, not {scores.dtype} {list(scores.shape)}")
    if (done is None) != (eos_id is None):
        raise ValueError("done and eos_id are given together")
    if done is not None:
        if done.dtype != torch.bool or done.shape != (B, K):
            raise ValueError(f"done must be bool {[B, K]}, not {done.dtype} {list(done.shape)}")
        if not 0 <= eos_id < V:
            raise ValueError(f"eos_id {eos_id} is outside the vocabulary of {V}")
    _together(dev, logits, scores, done)
    if not logits.is_cuda or B == 0:
        return _select_torch(logits, scores, done, eos_id)
    logits, scores = logits.contiguous(), scores.contiguous()
    done = None if done is None else done.contiguous()
    out = BeamStep(torch.empty_like(scores), torch.empty(B, K, dtype=torch.int64, device=dev), torch.empty(B, K, dtype=torch.int32, device=dev),
                   None if done is None else torch.empty_like(done))
    L = _lib.lib()
    work = torch.empty(L.axb_beam_select_words(B, K, V, _DT[logits.dtype]), dtype=torch.int32, device=dev)
    st = L.axb_beam_select(logits.data_ptr(), scores.data_ptr(), _lib.addr(done), -1 if done is None else eos_id, out.scores.data_ptr(),
                           out.tokens.data_ptr(), out.parents.data_ptr(), _lib.addr(out.done), work.data_ptr(), B, K, V, _DT[logits.dtype],
                           _lib.stream())
    _lib.check(st, "axb_beam_select")
    _lib.add_launches(1)
    return out


def _select_torch(logits, scores, done, eos_id):
    B, K, V = logits.shape
    x, score = logits.detach().double(), torch.where(scores < float("inf"), scores, float("-inf")).double()[..., None]
    value = score + (x - x.logsumexp(-1, keepdim=True))
    if done is not None:
        value = torch.where(done[..., None], torch.where(torch.arange(V, device=x.device) == eos_id, score, float("-inf")), value)
    value = value.masked_fill(value.isnan(), float("-inf")).reshape(B, K * V)
    value, at = value.sort(stable=True, dim=-1, descending=True)
    at = at[:, :K]
    parents, tokens = at // V, at % V
    ended = None if done is None else done.gather(1, parents) | (tokens == eos_id)
    return BeamStep(value[:, :K].float(), tokens, parents.int(), ended)
