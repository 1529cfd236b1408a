"""Memory that linear attention asks for on packed batches, and its refusals, without a device."""
import pytest
import torch

from rwkv_ops_b200 import _lib, _ops
from rwkv_ops_b200.build import build


@pytest.fixture(scope="module")
def lib():
    if not _ops.built():
        build()
    _ops.load()
    return _lib.load()


A = 0x1000      # a fake, 16-byte aligned address; never dereferenced because validation fails first
CODES = ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("code,dtype", CODES)
def test_packed_memory_is_that_of_the_tokens(lib, code, dtype, D):
    n, longest, H = 513, 32768, 32
    total = longest + 512 * 40
    state = H * D * D * 4
    need = lib.rwkvb200_linattn_packed_states_bytes(n, longest, total, H, D, code, 1)
    assert 0 < need <= (total // 64 + 2 * n) * state
    assert need * 20 < lib.rwkvb200_linattn_states_bytes(n, longest, H, D, code, 1)
    scratch = lib.rwkvb200_linattn_packed_workspace_bytes(n, longest, total, H, D, code, 1, 1)
    # gradients of the states (or, on tensor cores, what parts of sequences add to them: some of the device's CTAs' worth), decays, and sums of dw
    assert 0 < scratch <= (total // 64 + 2 * n) * state + (1 << 25)


@pytest.mark.parametrize("n,T,total,H,D", [(1, 1, 1, 1, 64), (2, 128, 200, 3, 64), (3, 129, 131, 2, 128), (8, 4096, 20000, 32, 64), (5, 1000, 4100, 7, 128),
                                           (700, 900, 5000, 2, 64), (4, 512, 2048, 1, 64)])
def test_shape_functions_of_packed_batches(lib, n, T, total, H, D):
    for code, dtype in CODES:
        need = lib.rwkvb200_linattn_packed_states_bytes(n, T, total, H, D, code, 1)
        assert _lib.linattn_states_bytes(n, T, H, D, dtype, total) == need
        assert need <= lib.rwkvb200_linattn_states_bytes(n, T, H, D, code, 1)      # (memory for the padded form is always enough)


def test_packed_refusals(lib):
    def fwd(sb, wb=1 << 40, n=50, T=1000, total=2000, H=3, D=64, dtype=0):
        return lib.rwkvb200_linattn_fwd(A, A, 0, A, A, None, 0, A, A, A, sb, A, wb, A, A, n, T, total, H, D, dtype, 0, None)

    def bwd(sb, wb=1 << 40, n=50, T=1000, total=2000, H=3, D=64, dtype=0):
        return lib.rwkvb200_linattn_bwd(A, A, 1, A, A, A, None, A, sb, A, A, A, A, None, A, wb, A, A, n, T, total, H, D, dtype, 0, None)

    for D, dtype in ((64, 0), (64, 1), (64, 2), (128, 1)):
        need = lib.rwkvb200_linattn_packed_states_bytes(50, 1000, 2000, 3, D, dtype, 1)
        assert fwd(need - 1, D=D, dtype=dtype) == -5 and bwd(need - 1, D=D, dtype=dtype) == -5
        scratch = lib.rwkvb200_linattn_packed_workspace_bytes(50, 1000, 2000, 3, D, dtype, 1, 1)
        assert scratch > 0 and bwd(need, scratch - 1, D=D, dtype=dtype) == -5
        # memory for the padded form means the padded form, which wants its workspace, too
        padded = lib.rwkvb200_linattn_states_bytes(50, 1000, 3, D, dtype, 1)
        wide = lib.rwkvb200_linattn_workspace_bytes(50, 1000, 2000, 3, D, dtype, 1, 1)
        assert bwd(padded, wide - 1, D=D, dtype=dtype) == -5
    assert lib.rwkvb200_linattn_packed_states_bytes(50, 1000, 0, 3, 64, 0, 1) == 0
    # too many blocks padded, not compact; and too many either way
    assert lib.rwkvb200_linattn_states_bytes(1 << 15, 1 << 20, 8, 64, 0, 1) == 0
    assert lib.rwkvb200_linattn_packed_states_bytes(1 << 15, 1 << 20, 1 << 21, 8, 64, 0, 1) > 0
    assert lib.rwkvb200_linattn_packed_states_bytes(1 << 15, 1 << 30, 1 << 30, 200, 64, 0, 1) == 0
