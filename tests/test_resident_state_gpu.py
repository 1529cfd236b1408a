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


@pytest.mark.parametrize("rwkv7", [False, True])
@pytest.mark.parametrize("n,dtype", [(1, torch.float32), (1, torch.bfloat16), (64, torch.bfloat16), (64, torch.float32)])
def test_a_state_is_made_once(n, dtype, rwkv7):
    """From one state for all, or of another type: no memory beside the state's own; and never a part of an autograd graph."""
    import rwkv_ops_b200 as ro
    B, H = 64, 8
    s = torch.randn(n, H, 64, 64, device="cuda", requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dec = (ro.Rwkv7DecodeState if rwkv7 else ro.LinearAttentionDecodeState)(B, H, state_dtype=dtype, initial_state=s)
    size = B * H * 4096 * dec.state.element_size()
    assert torch.cuda.max_memory_allocated() - before <= size + 4096
    assert not dec.state.requires_grad and dec.state.is_contiguous() and dec.state.data_ptr() != s.data_ptr()
    assert torch.equal(dec.state, s.detach().expand(B, H, 64, 64).to(dtype))
    dec.reorder(torch.tensor([[1, 0]] * 32, device="cuda"))
    assert torch.equal(dec.state, s.detach().expand(B, H, 64, 64).to(dtype).view(32, 2, H, 64, 64).flip(1).flatten(0, 1))
    strided = s.detach().transpose(2, 3)
    assert torch.equal((ro.Rwkv7DecodeState if rwkv7 else ro.LinearAttentionDecodeState)(B, H, initial_state=strided).state, strided.expand(B, H, 64, 64))
