"""Beam search over recurrent states: the selection of the best continuations (``beam_select``).

A step of beam search with a decode state (``Rwkv7DecodeState`` or ``LinearAttentionDecodeState``, ``groups * beams`` sequences)::

    scores, parents, tokens, finished = beam_select(logits, scores, finished=finished, eos=eos)
    state.reorder(parents)              # or state.step(..., parents=parents) with the next token

The state of a sequence is all that there is to its past, so following the beams is a permutation (with repetitions) of states, done in
place.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib, _ops

MAX_BEAMS = 32


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None, eos: Optional[int] = None):
    """The ``beams`` best continuations of every search, in one pass over the logits.

    ``logits``: ``[groups, beams, vocabulary]`` (float32, bfloat16 or float16, last dimension contiguous, any other strides); ``scores``:
    ``[groups, beams]``, the beams' summed log-probabilities (``-inf`` for a beam that does not exist yet).  Candidate ``(i, t)`` has the score
    ``scores[i] + log_softmax(logits[i])[t]``; candidates are compared in float64, equal ones go to the lower beam, then to the larger logit, then to the lower token.
    ``finished`` (bool, like ``scores``; needs ``eos``): such a beam goes on with ``eos`` alone, at the score it has.

    Returns ``(scores, parents, tokens)``, each ``[groups, beams]`` in descending order of scores (float32, int64, int64), and with ``eos``
    also ``finished`` (the parent had finished, or the token is ``eos``).  Logits that are NaN or ``+inf`` count as ``-inf``; where fewer than ``beams`` continuations are possible, impossible ones follow with score ``-inf``.  At most 32 beams.  Nothing is differentiated.
    """
    if finished is not None and eos is None:
        raise ValueError("finished needs eos")
    if eos is not None and eos < 0:
        raise ValueError(f"eos must be a token, got {eos}")
    try:
        best, parents, tokens, done = _ops.load().beam_select(logits, scores, finished, -1 if eos is None else int(eos))
    except Exception as e:
        _lib.require_cuda(logits, scores, finished)
        raise _ops.failed(e)
    return (best, parents, tokens) if eos is None else (best, parents, tokens, done)
