"""Tracing of the operators that are called as they are (steps on resident states, reordering, beam selection) and of packed linear attention, on
fake CUDA tensors: shapes, strides, symbols and refusals are the operators'."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import rwkv_ops_b200 as ro
from rwkv_ops_b200 import _ops
from rwkv_ops_b200.build import build
from test_tracing_cpu import _symbolic, _tokens


@pytest.fixture(scope="module", autouse=True)
def _operators():
    if not _ops.built():
        build()
    _ops.load()


def e(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def test_results_are_contiguous_whatever_the_strides():
    with FakeTensorMode():
        scores = e(3, 2).T
        got = ro.beam_select(e(2, 3, 50), scores, finished=e(3, 2, dtype=torch.bool).T, eos=4)
        assert [t.stride() for t in got] == [(3, 1)] * 4
        assert [t.dtype for t in got] == [torch.float32, torch.int64, torch.int64, torch.bool]
        for r in (e(4, 8, 64, dtype=torch.bfloat16).transpose(0, 1), e(8, 64, 4).transpose(1, 2), e(8, 4, 128)[..., ::2],
                  e(1, 8, 4, 64).transpose(0, 1)):
            o = ro.LinearAttentionDecodeState(8, 4).step(r, e(4), r, r)
            assert o.shape == r.shape and o.is_contiguous() and o.dtype == r.dtype
            o = ro.Rwkv7DecodeState(8, 4).step(r, r, r, r, r, r)
            assert o.shape == r.shape and o.is_contiguous() and o.dtype == r.dtype


def test_symbols_stay_symbols():
    mode, sizes, (logits,) = _tokens(1, (6, 4, 5000), torch.float32)
    with mode:
        assert all(all(_symbolic(t, (0, 1))) for t in ro.beam_select(logits, e(*sizes[:2]), eos=3))


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("grad", [False, True])
def test_packed_batches(dtype, D, grad):
    with FakeTensorMode():
        p = ro.PackedSequences.__new__(ro.PackedSequences)
        p.total_len, p.max_len, p.start, p.lens = 900, 300, e(5, dtype=torch.int32), e(5, dtype=torch.int32)
        r, k, v = (torch.empty(1, 900, 3, D, dtype=dtype, device="cuda", requires_grad=grad) for _ in range(3))
        w = torch.empty(3, device="cuda", requires_grad=grad)
        o, s = ro.linear_attention_varlen(r, w, k, v, p)
        assert o.shape == r.shape and o.dtype == dtype and s.shape == (5, 3, D, D) and s.dtype == torch.float32
        # (the autograd engine wants a device; the operator that it calls does not)
        g = _ops.load().linattn_bwd(r, w, k, v, p.start, p.lens, 300, None, o, s, torch.empty(0, dtype=torch.uint8, device="cuda"), False)
        assert [t.shape for t in g] == [t.shape for t in (r, w, k, v, s)]


class Search(torch.nn.Module):
    """A step of beam search: selection, and a step that follows it."""

    def forward(self, logits, scores, finished, r, w, k, v, state):
        best, parents, tokens, done = ro.beam_select(logits, scores, finished=finished, eos=2)
        o = _ops.load().linattn_step(r, w, k, v, state, parents)
        _ops.load().reorder_states(state, parents)
        return best, tokens, done, o


def test_export_of_a_search_step():
    with FakeTensorMode(), torch.no_grad():
        r, k, v = (e(6, 1, 4, 64, dtype=torch.bfloat16) for _ in range(3))
        args = (e(2, 3, 50), e(2, 3), e(2, 3, dtype=torch.bool), r, e(6, 1, 4), k, v, e(6, 4, 64, 64))
        program = torch.export.export(Search(), args)
    names = " ".join(str(n.target) for n in program.graph.nodes)
    assert all(f"rwkv_ops_b200.{n}" in names for n in ("beam_select", "linattn_step", "reorder_states"))


def test_wrong_arguments_raise():
    with FakeTensorMode():
        x, s, f = e(2, 3, 50), e(2, 3), e(2, 3, dtype=torch.bool)
        for bad in (lambda: ro.beam_select(x[0], s), lambda: ro.beam_select(x, s[:1]), lambda: ro.beam_select(x[..., :0], s),
                    lambda: ro.beam_select(x, s, eos=50), lambda: ro.beam_select(x, s, finished=f[:1], eos=3),
                    lambda: ro.beam_select(e(1, 33, 5), e(1, 33))):
            with pytest.raises(ValueError):
                bad()
        dec, r, w, p = ro.LinearAttentionDecodeState(2, 3), e(2, 3, 64), e(3), torch.empty(1, 2, dtype=torch.long, device="cuda")
        dec.step(r, w, r, r, parents=p)
        dec.reorder(p)
        for bad in (lambda: dec.step(r, w, r[:1], r), lambda: dec.step(r[:1], w, r[:1], r[:1]), lambda: dec.step(r, w[:2], r, r),
                    lambda: dec.step(r[..., :32], w, r[..., :32], r[..., :32]), lambda: dec.step(e(2, 2, 3, 64), w, e(2, 2, 3, 64), e(2, 2, 3, 64)),
                    lambda: dec.step(r, w, r, r, parents=p[0]), lambda: dec.step(r, w, r, r, parents=p.float()),
                    lambda: dec.reorder(p[:, :1]), lambda: ro.reorder_states(e(66, 4), torch.empty(2, 33, dtype=torch.long, device="cuda")),
                    lambda: ro.reorder_states(e(4, 3), torch.empty(2, 2, dtype=torch.long, device="cuda")),
                    lambda: ro.reorder_states(e(4, 8)[:, ::2], torch.empty(2, 2, dtype=torch.long, device="cuda")),
                    lambda: ro.Rwkv7DecodeState(2, 3).step(r, r, r, r, r, r[:1])):
            with pytest.raises(ValueError):
                bad()
