"""The torch operators of ``csrc/torch_ops.cpp``, loaded once, and their shape functions.

``load()`` returns the operator namespace (``torch.ops.rwkv_ops_b200``); it raises if one of the two libraries has
not been built.  ``failed(error)`` turns an operator's error into the exception the package documents.
"""
from __future__ import annotations

import os

import torch

from . import _lib
from ._lib import RwkvB200Error

OPS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "librwkv_ops_b200_torch.so")

_ops = None


def load():
    global _ops
    if _ops is None:
        _lib.load()      # the C ABI the operators call
        if not os.path.exists(OPS_PATH):
            raise RwkvB200Error(f"{OPS_PATH} not found. Build it with `python -m rwkv_ops_b200.build`; "
                                     "rwkv_ops_b200 has no eager fallback.")
        try:
            torch.ops.load_library(OPS_PATH)
        except OSError as e:
            raise RwkvB200Error(f"{OPS_PATH} does not load with torch {torch.__version__}; rebuild it with "
                                f"`python -m rwkv_ops_b200.build`: {e}") from e
        _register_fakes()
        _ops = torch.ops.rwkv_ops_b200
    return _ops


def built() -> bool:
    return os.path.exists(OPS_PATH) and os.path.exists(_lib.LIB_PATH)


def failed(error: Exception) -> Exception:
    """What to raise for an operator call that failed on valid arguments."""
    text = str(error)
    if type(error) is RuntimeError and text.startswith("rwkv_ops_b200 "):
        return RwkvB200Error(text.splitlines()[0])
    return error


def _register_fakes():
    fake = torch.library.register_fake

    def state(r, n, H, K):
        return r.new_empty((n, H, K, K), dtype=torch.float32)

    def tokens(r, n):
        return tuple(torch.empty_like(r) for _ in range(n))

    def kept(r, n):
        return r.new_empty((n,), dtype=torch.uint8)

    # The operators that are called as they are, without a composite one that checks and lays out before them: they refuse what their kernels'
    # hosts refuse, and what they return is contiguous, whatever the arguments' strides.
    def need(ok, text):
        if not ok:
            raise ValueError(text)

    def step_tokens(r, rest, state):
        B, H, V, D = state.shape
        need(r.device.type == "cuda" and state.device == r.device and all(x.device == r.device and x.shape == r.shape for x in rest),
             "token tensors must agree in shape and device")
        need(r.dim() in (3, 4) and r.shape[0] == B and r.shape[-2] == H and r.shape[-1] == D == V and (r.dim() == 3 or r.shape[1] == 1),
             f"expected token tensors [{B}, 1, {H}, {D}] or [{B}, {H}, {D}], got {tuple(r.shape)}")
        need(state.is_contiguous() and state.dtype in (torch.float32, torch.bfloat16), "expected a contiguous float32 or bfloat16 state")

    def beam_parents(parents, state):
        need(parents.dim() == 2 and parents.device == state.device and not parents.is_floating_point() and not parents.is_complex()
             and parents.numel() == state.shape[0] and 1 <= parents.shape[1] <= 32,
             f"parents must be [groups, beams], at most 32 beams and {state.shape[0]} in all, got {tuple(parents.shape)}")

    def dims(r, head_first):
        B, T, H, K = r.shape
        return (B, H, T, K) if head_first else (B, T, H, K)

    @fake("rwkv_ops_b200::rwkv7_fwd")
    def _(r, w, k, v, a, b, h0, head_first, algo, keep):
        B, T, H, K = dims(r, head_first)
        tiles = K == 64 and r.dtype == torch.bfloat16 and algo & 0xff != _lib.ALGO_RECURRENT
        n = 0 if not keep else _lib.rwkv7_kept_bytes(B, T, H) if tiles else _lib.rwkv7_states_bytes(B, T, H, K)
        return torch.empty_like(r), state(r, B, H, K), kept(r, n)

    @fake("rwkv_ops_b200::rwkv7_bwd")
    def _(r, w, k, v, a, b, h0, d_o, d_ht, k_, head_first, algo):
        B, T, H, K = dims(r, head_first)
        return (*tokens(r, 6), state(r, B, H, K))

    @fake("rwkv_ops_b200::rwkv7_decode_step")
    def _(r, w, k, v, a, b, state):
        step_tokens(r, (w, k, v, a, b), state)
        return r.new_empty(r.shape)

    @fake("rwkv_ops_b200::rwkv7_fwd_varlen")
    def _(r, w, k, v, a, b, seq_start, seq_len, max_len, h0, keep):
        H, n = r.shape[2], seq_start.numel()
        return torch.empty_like(r), state(r, n, H, 64), kept(r, _lib.rwkv7_kept_bytes(n, max_len, H) if keep else 0)

    @fake("rwkv_ops_b200::rwkv7_bwd_varlen")
    def _(r, w, k, v, a, b, seq_start, seq_len, max_len, h0, d_o, d_ht, k_):
        return (*tokens(r, 6), state(r, seq_start.numel(), r.shape[2], 64))

    @fake("rwkv_ops_b200::rwkv7_fused_fwd")
    def _(r, w_pre, k, v, kk_pre, a_pre, h0, keep):
        B, T, H, K = r.shape
        return torch.empty_like(r), state(r, B, H, K), kept(r, _lib.rwkv7_kept_bytes(B, T, H) if keep else 0)

    @fake("rwkv_ops_b200::rwkv7_fused_bwd")
    def _(r, w_pre, k, v, kk_pre, a_pre, h0, d_o, d_ht, k_):
        B, T, H, K = r.shape
        return (*tokens(r, 6), state(r, B, H, K))

    @fake("rwkv_ops_b200::wkv6_fwd")
    def _(r, k, v, w, u, s0, state_map, algo, keep):
        B, T, C = r.shape
        H, N = u.shape
        sT = state(r, B, H, N)
        return (torch.empty_like(r), sT.to(r.dtype) if algo & _lib.ALGO_TOKEN_STATES else sT,
                kept(r, _lib.wkv6_kept_bytes(B, T, H) if keep else 0))

    @fake("rwkv_ops_b200::wkv6_bwd")
    def _(r, k, v, w, u, s0, state_map, d_y, d_sT, k_, algo):
        return (*tokens(r, 4), torch.empty_like(u), state(r, r.shape[0], *u.shape))

    @fake("rwkv_ops_b200::wkv6_fwd_varlen")
    def _(r, k, v, w, u, seq_start, seq_len, max_len, s0, state_map, keep):
        H, N = u.shape
        n = seq_start.numel()
        return torch.empty_like(r), state(r, n, H, N), kept(r, _lib.wkv6_kept_bytes(n, max_len, H) if keep else 0)

    @fake("rwkv_ops_b200::wkv6_bwd_varlen")
    def _(r, k, v, w, u, seq_start, seq_len, max_len, s0, state_map, d_y, d_sT, k_):
        return (*tokens(r, 4), torch.empty_like(u), state(r, seq_start.numel(), *u.shape))

    @fake("rwkv_ops_b200::linattn_fwd")
    def _(r, w, k, v, seq_start, seq_len, max_len, h0, head_first, keep):
        B, T, H, D = dims(r, head_first)
        n, length, total = (B, T, None) if seq_start is None else (seq_start.numel(), max_len, T)
        return torch.empty_like(r), state(r, n, H, D), kept(r, _lib.linattn_states_bytes(n, length, H, D, r.dtype, total) if keep else 0)

    @fake("rwkv_ops_b200::linattn_bwd")
    def _(r, w, k, v, seq_start, seq_len, max_len, h0, d_o, d_ht, k_, head_first):
        B, T, H, D = dims(r, head_first)
        return (torch.empty_like(r), torch.empty_like(w), *tokens(r, 2), state(r, B if seq_start is None else seq_start.numel(), H, D))

    @fake("rwkv_ops_b200::linattn_step")
    def _(r, w, k, v, state, parents):
        step_tokens(r, (k, v), state)
        need(w.device == r.device and (w.dim() == 1 and w.shape[0] == r.shape[-2] or w.shape == r.shape[:-1]),
             f"w must be [{r.shape[-2]}] or one number per token and head, got {tuple(w.shape)}")
        need(r.shape[-1] in (64, 128), f"head size must be 64 or 128, got {r.shape[-1]}")
        if parents is not None:
            beam_parents(parents, state)
        return r.new_empty(r.shape)

    @fake("rwkv_ops_b200::reorder_states")
    def _(state, parents):
        need(state.device.type == "cuda" and state.dim() >= 1 and state.is_contiguous() and state.numel() > 0,
             f"expected a contiguous CUDA tensor of states, got {tuple(state.shape)}")
        row = state.numel() // state.shape[0] * state.element_size()
        need(row % 16 == 0, f"a state must be a multiple of 16 bytes, got {row}")
        beam_parents(parents, state)
        return None

    @fake("rwkv_ops_b200::beam_select")
    def _(logits, scores, finished, eos):
        need(logits.device.type == "cuda" and logits.dim() == 3 and logits.numel() > 0,
             f"expected logits [groups, beams, vocabulary], got {tuple(logits.shape)}")
        need(scores.device == logits.device and scores.shape == logits.shape[:2],
             f"scores must be {list(logits.shape[:2])}, got {tuple(scores.shape)}")
        need(logits.shape[1] <= 32 and logits.shape[2] <= 1 << 30, f"at most 32 beams and 2^30 tokens, got {tuple(logits.shape)}")
        need(eos < logits.shape[2] and (eos >= 0 or finished is None), f"eos must be a token, got {eos}")
        need(finished is None or (finished.device == logits.device and finished.shape == scores.shape), "finished must be like scores")
        return (*(scores.new_empty(scores.shape, dtype=t) for t in (torch.float32, torch.int64, torch.int64)),
                scores.new_empty(scores.shape if eos >= 0 else (0,), dtype=torch.bool))
