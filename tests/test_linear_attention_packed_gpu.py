"""Linear attention on packed batches, beyond what the operator's own ``cu_seqlens`` can say: rows of no sequence through the C interface."""
import pytest
import torch

import linear_attention_reference as ref

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {F32: 0, BF16: 1, F16: 2}
SENTINEL = 77.0


def sequences_alone(x, start, lens, n_state):
    """with_gradients() of each sequence of a packed batch; the results of all of them: tokens by sequence, states, dw per head summed."""
    parts = []
    for i, (s, n) in enumerate(zip(start, lens)):
        y = {q: x[q][:, s:s + n] if x[q].dim() > 1 else x[q] for q in ("r", "w", "k", "v", "d_o")}
        y["s0"] = None if not n_state else x["s0"][i:i + 1] if n_state > 1 else x["s0"]
        y["d_s"] = x["d_s"][i:i + 1]
        parts.append(ref.with_gradients(y))
    want = {q: torch.cat([p[q] for p in parts], 1) for q in ("o", "dr", "dk", "dv")}
    want["s"] = torch.cat([p["s"] for p in parts])
    want["dw"] = sum(p["dw"] for p in parts) if x["w"].dim() == 1 else torch.cat([p["dw"] for p in parts], 1)
    if n_state:
        want["ds0"] = torch.cat([p["ds0"] for p in parts])
    return want


@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 64), (F16, 64), (F32, 128), (BF16, 128)])
@pytest.mark.parametrize("w", ["head", "token"])
def test_rows_of_no_sequence(dtype, D, w):
    """Rows before, between and behind the sequences: whatever they and the workspace hold (NaN), nothing of it reaches a result, and no
    output is written there."""
    from rwkv_ops_b200 import _lib
    lib = _lib.load()
    start, lens, total, H, code = [3, 140, 161, 300], [130, 1, 64, 200], 517, 3, CODE[dtype]
    n = len(lens)
    x = ref.inputs(1, total, H, D, dtype=dtype, w=w, seed=31)
    g = torch.Generator().manual_seed(32)
    x["s0"], x["d_s"] = 0.1 * torch.randn(n, H, D, D, generator=g), 0.1 * torch.randn(n, H, D, D, generator=g)
    want = sequences_alone(x, start, lens, n)
    rows = torch.cat([torch.arange(s, s + m) for s, m in zip(start, lens)])
    outside = torch.ones(total, dtype=torch.bool)
    outside[rows] = False
    a = {}
    for q in ("r", "w", "k", "v", "d_o"):
        a[q] = x[q].clone()
        if a[q].dim() > 1:
            a[q][:, outside] = float("nan")
        a[q] = a[q].cuda()
    s0, d_s = x["s0"].cuda(), x["d_s"].cuda()
    at, ln = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (start, lens))
    nan = lambda size: torch.full((max(16, size),), 0xff, dtype=torch.uint8, device="cuda")
    out = {q: torch.full((1, total, H, D), SENTINEL, dtype=dtype, device="cuda") for q in ("o", "dr", "dk", "dv")}
    out["dw"] = torch.full(x["w"].shape, SENTINEL, device="cuda")
    out["s"], out["ds0"] = torch.empty(n, H, D, D, device="cuda"), torch.empty(n, H, D, D, device="cuda")
    p = lambda t: t.data_ptr()
    per_head, longest = int(w == "head"), max(lens)
    sizes = (n, longest, total, H, D, code)
    states = nan(lib.rwkvb200_linattn_states_bytes(n, longest, H, D, code, 1))
    ws = [nan(lib.rwkvb200_linattn_workspace_bytes(*sizes, per_head, backward)) for backward in (0, 1)]
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.rwkvb200_linattn_fwd(p(a["r"]), p(a["w"]), per_head, p(a["k"]), p(a["v"]), p(s0), n, p(out["o"]), p(out["s"]), p(states), states.numel(),
                                    p(ws[0]), ws[0].numel(), p(at), p(ln), n, longest, total, H, D, code, 0, stream) == 0
    assert lib.rwkvb200_linattn_bwd(p(a["r"]), p(a["w"]), per_head, p(a["k"]), p(a["v"]), p(a["d_o"]), p(d_s), p(states), states.numel(),
                                    p(out["dr"]), p(out["dw"]), p(out["dk"]), p(out["dv"]), p(out["ds0"]), p(ws[1]), ws[1].numel(), p(at), p(ln),
                                    n, longest, total, H, D, code, 0, stream) == 0
    for q in ("o", "dr", "dk", "dv") + (("dw",) if w == "token" else ()):
        assert (out[q][:, outside.cuda()] == SENTINEL).all(), q
        out[q] = out[q][:, rows.cuda()]
    ref.check(out, want, dtype)
