"""Forward-mode derivatives are refused by every operator that has a backward, with or without gradients switched on: a tangent is not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

import rwkv_ops_b200 as ro
from rwkv_ops_b200 import _ops
from rwkv_ops_b200.build import build


@pytest.fixture(scope="module", autouse=True)
def _operators():
    if not _ops.built():
        build()
    _ops.load()


def e(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def packed():
    p = ro.PackedSequences.__new__(ro.PackedSequences)
    p.total_len, p.max_len, p.start, p.lens = 8, 5, e(2, dtype=torch.int32), e(2, dtype=torch.int32)
    return p


CALLS = {
    "linear_attention": (lambda x: ro.linear_attention(x[0], x[1], x[2], x[3], initial_state=x[4]),
                         lambda: [e(1, 8, 2, 64), e(2), e(1, 8, 2, 64), e(1, 8, 2, 64), e(1, 2, 64, 64, dtype=torch.float32)]),
    "linear_attention_varlen": (lambda x: ro.linear_attention_varlen(x[0], x[1], x[2], x[3], packed()), lambda: [e(1, 8, 2, 64), e(2), e(1, 8, 2, 64), e(1, 8, 2, 64)]),
    "generalized_delta_rule": (lambda x: ro.generalized_delta_rule(*x), lambda: [e(1, 8, 2, 64) for _ in range(6)]),
    "generalized_delta_rule_varlen": (lambda x: ro.generalized_delta_rule_varlen(*x, packed()), lambda: [e(1, 8, 2, 64) for _ in range(6)]),
    "generalized_delta_rule_fused": (lambda x: ro.generalized_delta_rule_fused(*x), lambda: [e(1, 8, 2, 64) for _ in range(6)]),
    "RWKV6_OP": (lambda x: ro.RWKV6_OP(64, 8)(*x, with_state=True), lambda: [e(1, 8, 128) for _ in range(4)] + [e(2, 64)]),
    "wkv6_varlen": (lambda x: ro.wkv6_varlen(*x, packed()), lambda: [e(1, 8, 128) for _ in range(4)] + [e(2, 64)]),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name, grad):
    call, inputs = CALLS[name]
    with FakeTensorMode(), torch.set_grad_enabled(grad):
        call(inputs())
        for i in range(len(inputs())):
            with fwAD.dual_level():
                x = inputs()
                x[i] = fwAD.make_dual(x[i], torch.empty_like(x[i]))
                with pytest.raises(NotImplementedError):
                    call(x)
