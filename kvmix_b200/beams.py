"""Beam search's selection on the device: which tokens continue which beams.

``KVmixPagedCache.advance`` calls it and lets the cache's rows follow.  No upstream counterpart: upstream decodes greedily or samples.
"""
import ctypes as C
import functools
import struct
from typing import NamedTuple

import torch

from . import _lib, ops
from ._lib import check

_pack = struct.Struct("@Pq8P6iPQ").pack
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class BeamStep(NamedTuple):
    """The n best continuations of every request, best first -- ``scores`` fp32, ``beams`` (within the request) and ``tokens`` int32, [requests, n] each -- and
    the first of them that do not end, [requests, beams] each, which is what goes on."""
    scores: torch.Tensor
    beams: torch.Tensor
    tokens: torch.Tensor
    next_scores: torch.Tensor
    next_beams: torch.Tensor
    next_tokens: torch.Tensor


def beam_select(logits, scores, beams, n=None, ends=None):
    """The best continuations of every request over its beams and the vocabulary, in two launches that read the logits once.

    logits [requests * beams, vocabulary] fp16, bf16 or fp32, any row stride; scores fp32 [requests * beams], the beams' so far.  A continuation's score is
    scores[beam] + log_softmax(logits[beam])[token]; the ``n`` best of a request (None: twice the beams, or beams * (1 + number of ends) where that is more; at most 128, beams at
    most 64) come in order, equal ones by (beam, token).  ends: int32 tensor of tokens that end a sequence; n must leave ``beams`` others, so beams * (1 + number of ends)
    is at most 128 too: one end for 64 beams, 31 for four.  A thread's sum of exponentials is fp32 (terms
    to 2^-22 of themselves, vocabulary / 256 of them at most and some hundred in large calls of few rows), from there they are 64-bit; rows alike have sums alike, to the last bit, but two
    beams whose continuations lie within that of each other may come in either order.
    A beam offers -infinity everywhere where its score is not finite (a beam that is not there: -infinity), its logits hold a NaN or +infinity, or all of
    them are masked (-infinity)."""
    dev = logits.get_device()
    if dev < 0:
        raise RuntimeError("kvmix_b200 operators need CUDA tensors (there is no CPU path)")
    if logits.dim() != 2 or logits.dtype not in _TYPES:
        raise RuntimeError("beam_select takes logits [requests * beams, vocabulary], fp16, bf16 or fp32")
    rows, vocabulary = logits.shape
    if not 0 < beams <= _lib.MOST_BEAMS or rows % beams or not 0 < vocabulary < 1 << 31:
        raise RuntimeError(f"rows come in groups of `beams`, at most {_lib.MOST_BEAMS}")
    if scores.dtype is not torch.float32 or scores.numel() != rows or scores.get_device() != dev or not scores.is_contiguous():
        raise RuntimeError(f"scores must be contiguous float32 [{rows}] on cuda:{dev}")
    n_ends, at_ends = 0, 0
    if ends is not None:
        if ends.dtype is not torch.int32 or ends.dim() != 1 or ends.get_device() != dev or not ends.is_contiguous():
            raise RuntimeError(f"ends must be a contiguous int32 tensor on cuda:{dev}")
        n_ends, at_ends = ends.numel(), ends.data_ptr()
    n = _how_many(n, beams, n_ends, vocabulary)
    if logits.stride(1) != 1 and vocabulary > 1:
        logits = logits.contiguous()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _select(logits, scores, beams, n, n_ends, at_ends)
    return _select(logits, scores, beams, n, n_ends, at_ends)


def _how_many(n, beams, n_ends, vocabulary):
    all_of_them = beams * vocabulary
    least, most = min(beams * (1 + n_ends), all_of_them), min(all_of_them, _lib.MOST_BEST)
    if least > most:
        raise RuntimeError(f"{beams} beams and {n_ends} ends take the {least} best continuations: beams * (1 + number of ends) is at most {most}")
    n = min(max(2 * beams, least), most) if n is None else int(n)
    if not least <= n <= most:
        raise RuntimeError(f"n must be {least} to {most} for {beams} beams and {n_ends} ends")
    return n


@functools.lru_cache(maxsize=None)
def _workspace_bytes(requests, beams, vocabulary, kind, n, n_ends):
    assert struct.calcsize("@Pq8P6iPQ") == C.sizeof(_lib.BeamArgs)
    return _lib.lib().kvq_beam_select_workspace_bytes(_pack(*[0] * 10, requests, beams, vocabulary, kind, n, n_ends, 0, 0))


def _select(logits, scores, beams, n, n_ends, at_ends):
    (rows, vocabulary), kind = logits.shape, _TYPES[logits.dtype]
    requests = rows // beams
    best, going = scores.new_empty((requests, n)), scores.new_empty((requests, beams))
    best_beams, going_beams = torch.empty_like(best, dtype=torch.int32), torch.empty_like(going, dtype=torch.int32)
    best_tokens, going_tokens = torch.empty_like(best_beams), torch.empty_like(going_beams)
    if requests:
        need = _workspace_bytes(requests, beams, vocabulary, kind, n, n_ends)
        workspace = scores.new_empty((need + 3) // 4)
        a = _pack(logits.data_ptr(), logits.stride(0), scores.data_ptr(), at_ends, best.data_ptr(), best_beams.data_ptr(), best_tokens.data_ptr(), going.data_ptr(),
                  going_beams.data_ptr(), going_tokens.data_ptr(), requests, beams, vocabulary, kind, n, n_ends, workspace.data_ptr(), need)
        rc = _lib._lib.kvq_beam_select(a, ops.raw_stream())            # loaded: _workspace_bytes asked it
        if rc:
            check(rc)
        ops.LAUNCHES[0] += 2
    return BeamStep(best, best_beams, best_tokens, going, going_beams, going_tokens)
