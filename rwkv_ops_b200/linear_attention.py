"""Linear attention with a decay for each head.

Per (sequence, head), with ``S`` a matrix of value by key channels::

    S_t = exp(-exp(w_t)) S_{t-1} + v_t k_t^T        o_t = S_t r_t

The interface follows ``generalized_delta_rule``: ``w`` is the raw decay input, states are float32 ``[N, H, V, K]``, the output has
``r``'s dtype.  ``w`` is a number per head (``[H]``, a fixed or learned decay) or per token and head (``[B, T, H]``, a decay that depends on the
data), and is taken in float32 whatever the tokens' dtype.  Any decay is exact: nothing is divided by a product of decays, so
``w = -1e9`` leaves the state alone (padding) and a large ``w`` clears it (the start of another document).  Values that are not finite reach
no other sequence and no token before the chunk they are in (128 tokens for bfloat16 at head size 64, else 64), but may reach earlier ones of it.

``linear_attention`` is the operator of prompts and training (a chunked form, forward and backward), ``linear_attention_varlen`` the same
over sequences packed end to end, and ``LinearAttentionDecodeState`` the recurrent form for one token at a time.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib, _ops
from .varlen import PackedSequences, _pack

HEAD_SIZES = (64, 128)


def _check_tokens(r, w, k, v, initial_state, head_first):
    _lib.require_cuda(r, w, k, v, initial_state)
    if r.dim() != 4 or r.shape[-1] not in HEAD_SIZES:
        raise ValueError(f"expected 4-D token tensors with head size in {HEAD_SIZES}, got {tuple(r.shape)}")
    for name, x in (("k", k), ("v", v)):
        if x.shape != r.shape:
            raise ValueError(f"{name} has shape {tuple(x.shape)}, expected {tuple(r.shape)}")
    H = r.shape[1] if head_first else r.shape[2]
    if tuple(w.shape) not in ((H,), tuple(r.shape[:3])):
        raise ValueError(f"w must be [{H}] or {list(r.shape[:3])}, got {tuple(w.shape)}")
    return H


def _check_state(initial_state, n, H, D):
    if initial_state is not None and (initial_state.dim() != 4 or tuple(initial_state.shape[1:]) != (H, D, D)
                                      or initial_state.shape[0] not in (1, n)):
        raise ValueError(f"initial_state must be [{n} or 1, {H}, {D}, {D}], got {tuple(initial_state.shape)}")


def linear_attention(r, w, k, v, initial_state: Optional[torch.Tensor] = None, output_final_state: bool = True,
                     head_first: bool = False):
    """``r, k, v``: ``[B, T, H, D]`` (``[B, H, T, D]`` when ``head_first``) with head size ``D`` 64 or 128, any of float32 /
    bfloat16 / float16; ``w``: ``[H]`` or ``[B, T, H]`` (``[B, H, T]``).  ``initial_state``: float32 ``[N, H, D, D]`` with ``N == B`` or
    ``N == 1`` (broadcast), value index before key index.  Returns ``(o, final_state)`` or just ``o``.  Differentiable with
    respect to ``r, w, k, v`` and ``initial_state``.
    """
    try:
        o, ht = _ops.load().linear_attention(r, w, k, v, None, None, 0, initial_state, bool(head_first))
    except Exception as e:
        H = _check_tokens(r, w, k, v, initial_state, head_first)
        _check_state(initial_state, r.shape[0], H, r.shape[-1])
        raise _ops.failed(e)
    return (o, ht) if output_final_state else o


def linear_attention_varlen(r, w, k, v, cu_seqlens, initial_state: Optional[torch.Tensor] = None,
                            output_final_state: bool = True):
    """``linear_attention`` over sequences packed end to end: ``r, k, v`` ``[1, total_len, H, D]``, ``w`` ``[H]`` or ``[1, total_len, H]``,
    ``cu_seqlens`` ``n_seq + 1`` increasing integers from 0 to ``total_len`` (tensor, list or ``PackedSequences``), ``initial_state`` float32
    ``[n_seq or 1, H, D, D]``.  Returns ``(o, final_state)`` with one state per sequence, or just ``o``.
    """
    def check():
        H = _check_tokens(r, w, k, v, initial_state, False)
        if r.shape[0] != 1:
            raise ValueError(f"expected packed token tensors [1, total_len, H, D], got {tuple(r.shape)}")
        if isinstance(cu_seqlens, PackedSequences) and (cu_seqlens.total_len != r.shape[1] or cu_seqlens.start.device != r.device):
            raise ValueError("the PackedSequences object was made for another token count or device")
        return H

    try:
        if isinstance(cu_seqlens, PackedSequences) and r.dim() == 4 and cu_seqlens.total_len == r.shape[1] \
                and cu_seqlens.start.device == r.device:
            p = cu_seqlens
        else:
            check()
            p = cu_seqlens if isinstance(cu_seqlens, PackedSequences) else _pack(cu_seqlens, r.shape[1], r.device)
        o, ht = _ops.load().linear_attention(r, w, k, v, p.start, p.lens, p.max_len, initial_state, False)
    except Exception as e:
        H = check()
        p = cu_seqlens if isinstance(cu_seqlens, PackedSequences) else _pack(cu_seqlens, r.shape[1], r.device)
        _check_state(initial_state, p.start.numel(), H, r.shape[-1])
        raise _ops.failed(e)
    return (o, ht) if output_final_state else o


class LinearAttentionDecodeState:
    """State of ``batch`` sequences x ``heads`` heads for single-token steps, kept in place on the device.

    ``state`` is ``[batch, heads, D, D]`` (value index before key index, the layout of the operator's ``final_state``), float32 or
    bfloat16.  ``step`` takes ``r, k, v`` as ``[batch, 1, heads, D]`` or ``[batch, heads, D]`` and ``w`` as ``[heads]`` or one number per token
    and head, and returns ``o`` shaped like ``r``.

    Beam search: the sequences are ``groups * beams``, the beams of a search next to each other.  With ``parents`` (``[groups, beams]``, what
    ``beam_select`` returns) beam ``j`` of a search goes on from the state that beam ``parents[j]`` of that search had: the step reads it from there, so the
    reordering costs nothing.  ``reorder`` does it alone.  At most 32 beams; entries outside the search are clamped.
    Steps are not differentiated.
    """

    def __init__(self, batch: int, heads: int, *, head_size: int = 64, state_dtype: torch.dtype = torch.float32, device="cuda",
                 initial_state: Optional[torch.Tensor] = None):
        if state_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("state_dtype must be float32 or bfloat16")
        if head_size not in HEAD_SIZES:
            raise ValueError(f"head_size must be in {HEAD_SIZES}, got {head_size}")
        shape = (batch, heads, head_size, head_size)
        if initial_state is not None:
            _lib.require_cuda(initial_state)
            _check_state(initial_state, batch, heads, head_size)
            self.state = torch.empty(shape, dtype=state_dtype, device=initial_state.device)
            self.state.copy_(initial_state.detach())      # (one state may serve all sequences)
        else:
            self.state = torch.zeros(shape, dtype=state_dtype, device=device)
        if not self.state.is_cuda:
            raise _lib.RwkvB200Error("LinearAttentionDecodeState lives on a CUDA device; there is no CPU fallback.")

    def _check_args(self, r, w, k, v, parents):
        B, H, _, D = self.state.shape
        if tuple(r.shape) not in ((B, 1, H, D), (B, H, D)):
            raise ValueError(f"expected token tensors [{B}, 1, {H}, {D}] or [{B}, {H}, {D}], got {tuple(r.shape)}")
        for name, x in (("k", k), ("v", v)):
            if x.shape != r.shape:
                raise ValueError(f"{name} has shape {tuple(x.shape)}, expected {tuple(r.shape)}")
        if tuple(w.shape) not in ((H,), tuple(r.shape[:-1])):
            raise ValueError(f"w must be [{H}] or {list(r.shape[:-1])}, got {tuple(w.shape)}")
        _lib.require_cuda(r, w, k, v, self.state, parents)

    def step(self, r, w, k, v, parents: Optional[torch.Tensor] = None):
        try:
            return _ops.load().linattn_step(r, w, k, v, self.state, parents)
        except Exception as e:
            self._check_args(r, w, k, v, parents)
            raise _ops.failed(e)

    def reorder(self, parents: torch.Tensor) -> None:
        """Sequence ``j`` of each search takes the state of sequence ``parents[j]`` of that search; ``parents`` ``[groups, beams]``."""
        reorder_states(self.state, parents)

    def final_state(self) -> torch.Tensor:
        """The state as the operator would return it (float32 copy)."""
        return self.state.to(torch.float32)


def reorder_states(state: torch.Tensor, parents: torch.Tensor) -> torch.Tensor:
    """Reorder the rows of ``state`` (``[groups * beams, ...]``, contiguous, rows a multiple of 16 bytes) in place: row ``j`` of each group becomes what
    row ``parents[group, j]`` of the group was.  No second buffer is used, rows that stay are not touched.  At most 32 beams; entries
    outside the group are clamped.  Returns ``state``.
    """
    try:
        _ops.load().reorder_states(state, parents)
    except Exception as e:
        _lib.require_cuda(state, parents)
        raise _ops.failed(e)
    return state
