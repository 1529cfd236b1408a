"""What the precision of linear attention is claimed to be, where a coarser one would show: single products alone, and float32 results."""
import pytest
import torch

import linear_attention_reference as ref

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("B,T,H", [(1, 128, 2), (2, 300, 3), (1, 1500, 1)])
def test_gradients_that_come_from_the_state_alone(B, T, H):
    """Without a gradient of the outputs dv = D dS k and dk = D dS^T v, D the decay behind a token.  dS meets k and v in two bfloat16 parts, 2^-17 of each
    of its numbers at most; the result is rounded once, half a step, 2^-8 of it."""
    import rwkv_ops_b200 as ro
    x = ref.inputs(B, T, H, dtype=BF16, seed=41, w_mean=-5.0)
    a = {q: x[q].cuda().requires_grad_(True) for q in "rwkv"}
    o, s = ro.linear_attention(a["r"], a["w"], a["k"], a["v"])
    dv, dk = torch.autograd.grad((o, s), (a["v"], a["k"]), (torch.zeros_like(o), x["d_s"].cuda()))
    g = -torch.exp(x["w"].double())
    D = torch.exp(g.flip(1).cumsum(1).flip(1) - g)[..., None]
    dS = x["d_s"].double()
    for got, spec, t in ((dv, "bhvk,bthk->bthv", x["k"].double()), (dk, "bhvk,bthv->bthk", x["v"].double())):
        want, size = D * torch.einsum(spec, dS, t), D * torch.einsum(spec, dS.abs(), t.abs())
        # (2^-17 for the two parts, and as much again for float32 sums and decays: 64 terms of 2^-24, exponentials of 2^-22)
        off = (got.double().cpu() - want).abs() - 2.0 ** -8 * want.abs() - 2.0 ** -16 * size
        assert float(off.max()) <= 0, float((off / size).max())
