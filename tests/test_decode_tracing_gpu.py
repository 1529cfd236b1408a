"""The shape functions of the operators that are called as they are, against the operators: sizes, strides, types and which arguments change."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def check(op, *args):
    torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


def test_shape_functions_are_the_operators():
    from rwkv_ops_b200 import _ops
    ops, dev = _ops.load(), "cuda"
    g = torch.Generator(device=dev).manual_seed(1)
    r = torch.randn(4, 6, 64, generator=g, device=dev).transpose(0, 1)
    state = torch.randn(6, 4, 64, 64, generator=g, device=dev)
    parents = torch.tensor([[0, 0, 1], [2, 1, 0]], device=dev)
    for x in (r, r.bfloat16(), r.double(), r[:, None].expand(6, 1, 4, 64)):
        check(ops.linattn_step.default, x, torch.zeros(4, device=dev), x, x, state.clone(), parents)
        check(ops.linattn_step.default, x, x[..., 0], x, x, state.bfloat16(), None)
        check(ops.rwkv7_decode_step.default, x, x, x, x, x, x, state.clone())
    check(ops.reorder_states.default, state.clone(), parents)
    logits, scores = torch.randn(2, 3, 100, generator=g, device=dev), torch.zeros(3, 2, device=dev).T
    check(ops.beam_select.default, logits, scores, None, -1)
    check(ops.beam_select.default, logits.half(), scores, scores > 0, 7)
    check(ops.beam_select.default, logits.transpose(0, 1).transpose(0, 1)[..., ::2], scores.double(), scores < 1, 7)
