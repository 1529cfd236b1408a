"""Host side of linear attention and of beam search: refusals before anything is launched, sizes, signatures, tracing, and the definition that the
GPU tests compare with."""
import inspect

import pytest
import torch

import linear_attention_reference as ref
import rwkv_ops_b200 as ro
from rwkv_ops_b200 import _lib, _ops
from rwkv_ops_b200.build import build
from test_tracing_cpu import _symbolic, _tokens


@pytest.fixture(scope="module")
def lib():
    if not _ops.built():
        build()
    _ops.load()
    return _lib.load()


A = 0x1000      # a fake, 16-byte aligned address; never dereferenced because validation fails first


def test_forward_and_backward_refuse(lib):
    def fwd(r=A, w=A, k=A, v=A, h0=None, n_state=0, o=A, ht=A, states=A, sb=1 << 40, ws=A, wb=1 << 40, start=None, lens=None, n=2, T=100, total=0,
            H=3, D=64, dtype=0, head_first=0):
        return lib.rwkvb200_linattn_fwd(r, w, 0, k, v, h0, n_state, o, ht, states, sb, ws, wb, start, lens, n, T, total, H, D, dtype, head_first, None)

    def bwd(d_o=A, states=A, sb=1 << 40, ws=A, wb=1 << 40, dr=A, start=None, lens=None, n=2, T=100, total=0, D=64, dtype=0, head_first=0, per_head=0):
        return lib.rwkvb200_linattn_bwd(A, A, per_head, A, A, d_o, None, states, sb, dr, A, A, A, None, ws, wb, start, lens, n, T, total, 3, D, dtype,
                                        head_first, None)

    assert fwd(n=0) == -1 and fwd(T=0) == -1 and fwd(H=0) == -1
    assert fwd(D=32) == -6 and fwd(dtype=7) == -2
    assert fwd(k=None) == -4 and fwd(r=None) == -4 and fwd(o=None, states=None) == -4
    assert fwd(v=A + 8) == -3 and fwd(states=A + 4) == -3
    assert fwd(h0=A, n_state=3) == -1 and fwd(n_state=1) == -4
    assert fwd(start=A) == -4 and fwd(lens=A) == -4
    assert fwd(start=A, lens=A, total=0) == -1 and fwd(start=A, lens=A, total=200, head_first=1) == -1
    assert fwd(n=1 << 20, H=1 << 10) == -9 and fwd(n=1 << 13, H=1 << 12, T=1 << 20) == -9
    for dtype in (0, 1, 2):
        need = lib.rwkvb200_linattn_states_bytes(2, 100, 3, 64, dtype, 1)
        assert need > 0 and fwd(dtype=dtype, sb=need - 1) == -5
        assert bwd(dtype=dtype, sb=need - 1) == -5
        for per_head in (0, 1):
            scratch = lib.rwkvb200_linattn_workspace_bytes(2, 100, 0, 3, 64, dtype, per_head, 1)
            if scratch:
                assert bwd(dtype=dtype, per_head=per_head, wb=scratch - 1) == -5 and bwd(dtype=dtype, per_head=per_head, ws=None) == -5
    # a bfloat16 forward that leaves nothing for a backward needs no memory for states
    assert lib.rwkvb200_linattn_states_bytes(2, 100, 3, 64, 1, 0) == 0
    assert bwd(d_o=None) == -4 and bwd(states=None) == -4 and bwd(dr=A + 2) == -3 and bwd(D=96) == -6


def test_step_reorder_and_selection_refuse(lib):
    step = lib.rwkvb200_linattn_step
    assert step(A, A, 0, A, A, A, 0, A, None, 0, 1, 3, 64, 0, None) == -1
    assert step(A, A, 0, A, A, A, 2, A, None, 2, 1, 3, 64, 0, None) == -2
    assert step(A, A, 0, A, A, A, 0, A, None, 2, 1, 3, 96, 0, None) == -6
    assert step(A, A, 0, A, A, None, 0, A, None, 2, 1, 3, 64, 0, None) == -4
    assert step(A + 2, A, 0, A, A, A, 0, A, None, 2, 1, 3, 64, 1, None) == -3
    assert step(A, A, 0, A, A, A, 0, A, A, 2, 33, 3, 64, 0, None) == -9
    reorder = lib.rwkvb200_reorder_states
    assert reorder(A, A, 0, 2, 64, None) == -1 and reorder(A, A, 2, 2, 8, None) == -1 and reorder(A, A, 2, 2, 0, None) == -1
    assert reorder(None, A, 2, 2, 64, None) == -4 and reorder(A, None, 2, 2, 64, None) == -4 and reorder(A + 8, A, 2, 2, 64, None) == -3
    assert reorder(A, A, 2, 33, 64, None) == -9
    assert reorder(A, A, 2, 1, 64, None) == 0      # a beam alone: nothing to do
    select = lib.rwkvb200_beam_select

    def sel(x=A, dtype=0, s=A, f=None, eos=-1, fo=None, g=2, w=3, v=50, st=(150, 50)):
        return select(x, dtype, *st, s, f, eos, A, A, A, fo, g, w, v, None)

    assert sel(g=0) == -1 and sel(w=0) == -1 and sel(v=0) == -1 and sel(st=(-1, 50)) == -1
    assert sel(eos=50) == -1 and sel(f=A) == -1 and sel(fo=A) == -1
    assert sel(dtype=5) == -2 and sel(x=None) == -4 and sel(s=None) == -4
    assert sel(x=A + 2) == -3 and sel(x=A + 1, dtype=1) == -3 and sel(w=33) == -9


def test_sizes_of_the_shape_functions(lib):
    for n, T, H, D in [(1, 1, 1, 64), (2, 128, 3, 64), (3, 129, 2, 128), (8, 4096, 32, 64), (5, 1000, 7, 128)]:
        for code, dtype in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
            assert _lib.linattn_states_bytes(n, T, H, D, dtype) == lib.rwkvb200_linattn_states_bytes(n, T, H, D, code, 1)


def test_cpu_tensors_are_refused(lib):
    x, w = torch.zeros(1, 4, 2, 64), torch.zeros(2)
    for call in (lambda: ro.linear_attention(x, w, x, x), lambda: ro.linear_attention_varlen(x, w, x, x, [0, 4]),
                 lambda: ro.LinearAttentionDecodeState(1, 2, device="cpu"), lambda: ro.LinearAttentionDecodeState(1, 2, initial_state=torch.zeros(1, 2, 64, 64)),
                 lambda: ro.reorder_states(torch.zeros(4, 4), torch.zeros(1, 4, dtype=torch.long)),
                 lambda: ro.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2))):
        with pytest.raises(_lib.RwkvB200Error):
            call()
    with pytest.raises(ValueError):
        ro.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2), finished=torch.zeros(1, 2, dtype=torch.bool))


def test_signatures():
    def names(f):
        return list(inspect.signature(f).parameters)

    assert names(ro.linear_attention) == ["r", "w", "k", "v", "initial_state", "output_final_state", "head_first"]
    assert names(ro.linear_attention_varlen) == ["r", "w", "k", "v", "cu_seqlens", "initial_state", "output_final_state"]
    assert names(ro.LinearAttentionDecodeState.step) == ["self", "r", "w", "k", "v", "parents"]
    assert names(ro.beam_select) == ["logits", "scores", "finished", "eos"]
    assert names(ro.reorder_states) == ["state", "parents"] and names(ro.Rwkv7DecodeState.reorder) == ["self", "parents"]
    for name in ("linear_attention", "linear_attention_varlen", "LinearAttentionDecodeState", "reorder_states", "beam_select"):
        assert name in ro.__all__


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("grad", [False, True])
def test_symbolic_sizes_stay_symbols(lib, dtype, D, grad):
    mode, sizes, x = _tokens(3, (2, 100, 3, D), dtype)
    with mode, torch.set_grad_enabled(grad):
        if grad:
            for t in x:
                t.requires_grad_(True)
        for w in (torch.empty(3, device="cuda"), torch.empty(*sizes[:3], device="cuda")):
            for state in (None, torch.empty(1, 3, D, D, device="cuda"), torch.empty(sizes[0], 3, D, D, device="cuda")):
                o, s = ro.linear_attention(x[0], w, x[1], x[2], initial_state=state)
                assert all(_symbolic(o, (0, 1))) and all(_symbolic(s, (0,)))


def test_the_definitions_agree_with_themselves():
    """Two halves of a sequence are the whole; a beam selection by sorting all candidates is one by torch's softmax."""
    x = ref.inputs(2, 12, 2, 8, n_state=2, seed=3)
    a = [x[n] for n in "rwkv"]
    o, s = ref.linear_attention(*a, initial_state=x["s0"])
    o1, s1 = ref.linear_attention(*[t[:, :5] for t in a], initial_state=x["s0"])
    o2, s2 = ref.linear_attention(*[t[:, 5:] for t in a], initial_state=s1)
    assert torch.allclose(torch.cat([o1, o2], 1), o, rtol=1e-12, atol=1e-12) and torch.allclose(s2, s, rtol=1e-12, atol=1e-12)
    g = torch.Generator().manual_seed(4)
    logits, scores = torch.randn(3, 4, 11, generator=g), torch.randn(3, 4, generator=g)
    best, parents, tokens = ref.beam_select(logits, scores)
    want = (logits.double().log_softmax(-1) + scores.double()[..., None]).flatten(1).topk(4)
    assert torch.allclose(best, want.values, rtol=1e-12) and torch.equal(parents * 11 + tokens, want.indices)
