"""Resident states of the decode steps: states of another shape are refused, and the first one is made without a second copy."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2, 3, 32, 64), (2, 3, 64, 32), (2, 3, 1, 64), (2, 3, 64), (2, 3, 64, 64, 1), (2, 3, 128, 64)])
def test_states_of_another_shape(shape):
    """(The steps take the tokens' head size for both of a state's last sizes.)"""
    import rwkv_ops_b200 as ro
    r, w = torch.zeros(2, 3, 64, device="cuda"), torch.zeros(3, device="cuda")
    for dec, args in ((ro.LinearAttentionDecodeState(2, 3), (r, w, r, r)), (ro.Rwkv7DecodeState(2, 3), (r,) * 6)):
        dec.step(*args)
        dec.state = torch.zeros(shape, device="cuda")
        with pytest.raises(ValueError):
            dec.step(*args)
