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
@pytest.mark.parametrize("start,lens,total,compact", [
    ([3, 140, 161, 300], [130, 1, 64, 200], 517, False),
    ([300, 161, 3, 140], [200, 64, 130, 1], 517, False),                           # in any order
    ([3, 700, 705, 706, 771], [650, 3, 1, 64, 129], 920, True),                    # the chunks' states one behind another
    ([0, 1, 2, 3, 4, 5, 6], [1, 1, 1, 1, 1, 1, 514], 520, True),
    ([128 + 2 * i for i in range(40)] + [250], [1 + i % 2 for i in range(40)] + [300], 550, True),      # (more than a warp looks through at once)
])
def test_rows_of_no_sequence(dtype, D, w, start, lens, total, compact):
    """Rows before, between and behind the sequences: whatever they and the workspace hold (NaN), nothing of it reaches a result, and no
    output is written there."""
    from rwkv_ops_b200 import _lib
    lib = _lib.load()
    H, code = 3, CODE[dtype]
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
    if compact:
        need, padded = lib.rwkvb200_linattn_packed_states_bytes(*sizes, 1), lib.rwkvb200_linattn_states_bytes(n, longest, H, D, code, 1)
        assert need < padded
        states = nan(need)
        ws = [nan(lib.rwkvb200_linattn_packed_workspace_bytes(*sizes, per_head, backward)) for backward in (0, 1)]
    else:
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


@pytest.mark.parametrize("dtype,D,w,n_short", [(BF16, 64, "head", 300), (BF16, 64, "token", 700), (F32, 64, "head", 300), (F16, 64, "token", 1100),
                                               (BF16, 128, "head", 40)])
@pytest.mark.parametrize("keep", [True, False])
def test_one_long_sequence_among_many_short_ones(dtype, D, w, n_short, keep, monkeypatch):
    """What a packed batch is, and that it takes the memory of its tokens: states of some 64 or 128 tokens each and one or two more to a sequence, not the
    longest sequence's for every one."""
    import rwkv_ops_b200 as ro
    if not keep:
        monkeypatch.setenv("RWKV_OPS_B200_KEEP_LIMIT_MB", "0")
    g = torch.Generator().manual_seed(33)
    H = 2
    lens = torch.randint(1, 12, (n_short,), generator=g).tolist()
    lens[n_short // 3] = 1500 if D == 64 else 700
    cu = torch.tensor([0] + lens).cumsum(0)
    T, n = int(cu[-1]), len(lens)
    x = ref.inputs(1, T, H, D, dtype=dtype, w=w, seed=34)
    x["s0"], x["d_s"] = 0.1 * torch.randn(1, H, D, D, generator=g), 0.1 * torch.randn(n, H, D, D, generator=g)
    want = sequences_alone(x, cu[:-1].tolist(), lens, 1)
    want["ds0"] = want["ds0"].sum(0, keepdim=True)
    a = {q: x[q].cuda().requires_grad_(True) for q in ("r", "w", "k", "v", "s0")}
    d_o, d_s = x["d_o"].cuda(), x["d_s"].cuda()
    p = ro.PackedSequences(cu, "cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    o, s = ro.linear_attention_varlen(a["r"], a["w"], a["k"], a["v"], p, initial_state=a["s0"])
    grads = torch.autograd.grad((o, s), list(a.values()), (d_o, d_s))
    used = torch.cuda.max_memory_allocated() - before
    C, state, tokens = 64, H * D * D * 4, T * H * D * (torch.finfo(dtype).bits // 8)
    # states and their gradients, o, s, the four token gradients and what the engine copies of them, dh0 and its sum, small things
    assert used <= 2 * (T // C + 2 * n) * state + 3 * n * state + 8 * tokens + (1 << 22), (used, T // C, n, state)
    got = dict(zip(["o", "s", "dr", "dw", "dk", "dv", "ds0"], [o, s, *grads]))
    ref.check(got, want, dtype)


@pytest.mark.parametrize("n", [63, 64, 65, 256, 257, 513])
def test_as_many_sequences_as_are_put_in_order_and_more(n):
    """The order in which sequences are worked on is not seen: together they are what two halves of them are, and each is its definition."""
    import rwkv_ops_b200 as ro
    g = torch.Generator(device="cuda").manual_seed(n)
    H = 2
    lens = torch.randint(1, 300, (n,), generator=g, device="cuda").cpu()
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
    T = int(cu[-1])
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = [rand(1, T, H, 64).to(BF16), -3 + rand(1, T, H), rand(1, T, H, 64).to(BF16) / 8, rand(1, T, H, 64).to(BF16)]
    d_o, d_s = rand(1, T, H, 64).to(BF16), 0.1 * rand(n, H, 64, 64)

    def call(a, b):      # sequences a .. b - 1
        cut = slice(int(cu[a]), int(cu[b]))
        y = [t[:, cut].contiguous().requires_grad_(True) for t in x]
        o, s = ro.linear_attention_varlen(*y, cu[a:b + 1] - cu[a])
        return [o.detach(), *torch.autograd.grad((o, s), y, (d_o[:, cut].contiguous(), d_s[a:b].contiguous()))], s.detach()

    tokens, states = call(0, n)
    k = n // 2
    parts = [call(0, k), call(k, n)]
    # (the halves may be cut into other stretches, whose starts are summed in another order: float32's last bits)
    for i, t in enumerate(tokens):
        want = torch.cat([p[0][i] for p in parts], 1)
        tol = ref.tolerance("dw" if i == 2 else "o", BF16)
        assert float((t.double() - want.double()).norm() / want.double().norm()) <= tol
    assert float((states - torch.cat([p[1] for p in parts])).norm() / states.norm()) <= ref.tolerance("s", F32)
    for i in range(0, n, max(1, n // 7)):      # and single ones against the definition
        cut = slice(int(cu[i]), int(cu[i + 1]))
        y = {q: t[:, cut].cpu() for q, t in zip("rwkv", x)}
        y.update(s0=None, d_o=d_o[:, cut].cpu(), d_s=d_s[i:i + 1].cpu())
        got = dict(zip(["o", "dr", "dw", "dk", "dv"], [t[:, cut] for t in tokens]))
        ref.check({**got, "s": states[i:i + 1]}, ref.with_gradients(y), BF16)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F32, 64), (F16, 128)])
@pytest.mark.parametrize("name", ["r", "w", "k", "v", "d_o", "d_s", "s0"])
def test_a_sequence_leaves_its_neighbours_alone(name, dtype, D):
    """NaN in any argument of one sequence, which begins and ends inside its neighbours' chunks, changes no bit of theirs."""
    import rwkv_ops_b200 as ro
    cu, H = [0, 70, 131, 195, 452], 2
    x = ref.inputs(1, cu[-1], H, D, dtype=dtype, seed=35)
    g = torch.Generator().manual_seed(36)
    x["s0"], x["d_s"] = 0.1 * torch.randn(4, H, D, D, generator=g), 0.1 * torch.randn(4, H, D, D, generator=g)

    def call(x):
        a = {q: x[q].cuda().requires_grad_(True) for q in ("r", "w", "k", "v", "s0")}
        o, s = ro.linear_attention_varlen(a["r"], a["w"], a["k"], a["v"], cu, initial_state=a["s0"])
        return [o, s, *torch.autograd.grad((o, s), list(a.values()), (x["d_o"].cuda(), x["d_s"].cuda()))]

    bad = dict(x)
    bad[name] = x[name].clone()
    if name in ("s0", "d_s"):
        bad[name][2] = float("nan")
    else:
        bad[name][:, 131:195] = float("nan")
    for p, q in zip(call(x), call(bad)):
        if p.shape[0] == 4:
            assert torch.equal(p[[0, 1, 3]], q[[0, 1, 3]])
        else:
            assert torch.equal(p[:, :131], q[:, :131]) and torch.equal(p[:, 195:], q[:, 195:])


@pytest.mark.parametrize("compact", [False, True])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 64), (F16, 128)])
def test_sequences_without_tokens(dtype, D, compact):
    """Through the C interface a sequence may be empty: its last state is its first one, and so are their gradients."""
    from rwkv_ops_b200 import _lib
    lib = _lib.load()
    start, lens, total, H, code = [0, 0, 400, 400, 401, 402, 402], [0, 400, 0, 1, 1, 0, 0], 402, 2, CODE[dtype]
    n, full = len(lens), [i for i, m in enumerate(lens) if m]
    x = ref.inputs(1, total, H, D, dtype=dtype, w="head", seed=37)
    g = torch.Generator().manual_seed(38)
    x["s0"], x["d_s"] = 0.1 * torch.randn(n, H, D, D, generator=g), 0.1 * torch.randn(n, H, D, D, generator=g)
    want = sequences_alone({**x, "s0": x["s0"][full], "d_s": x["d_s"][full]}, [start[i] for i in full], [lens[i] for i in full], len(full))
    a = {q: x[q].cuda() for q in ("r", "w", "k", "v", "d_o", "s0", "d_s")}
    at, ln = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (start, lens))
    nan = lambda size: torch.full((max(16, size),), 0xff, dtype=torch.uint8, device="cuda")
    out = {q: torch.empty(1, total, H, D, dtype=dtype, device="cuda") for q in ("o", "dr", "dk", "dv")}
    out["dw"], out["s"], out["ds0"] = torch.empty(H, device="cuda"), torch.empty(n, H, D, D, device="cuda"), torch.empty(n, H, D, D, device="cuda")
    p, sizes = (lambda t: t.data_ptr()), (n, max(lens), total, H, D, code)
    if compact:
        states = nan(lib.rwkvb200_linattn_packed_states_bytes(*sizes, 1))
        ws = [nan(lib.rwkvb200_linattn_packed_workspace_bytes(*sizes, 1, backward)) for backward in (0, 1)]
    else:
        states = nan(lib.rwkvb200_linattn_states_bytes(n, max(lens), H, D, code, 1))
        ws = [nan(lib.rwkvb200_linattn_workspace_bytes(*sizes, 1, backward)) for backward in (0, 1)]
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.rwkvb200_linattn_fwd(p(a["r"]), p(a["w"]), 1, p(a["k"]), p(a["v"]), p(a["s0"]), n, p(out["o"]), p(out["s"]), p(states), states.numel(),
                                    p(ws[0]), ws[0].numel(), p(at), p(ln), n, max(lens), total, H, D, code, 0, stream) == 0
    assert lib.rwkvb200_linattn_bwd(p(a["r"]), p(a["w"]), 1, p(a["k"]), p(a["v"]), p(a["d_o"]), p(a["d_s"]), p(states), states.numel(), p(out["dr"]),
                                    p(out["dw"]), p(out["dk"]), p(out["dv"]), p(out["ds0"]), p(ws[1]), ws[1].numel(), p(at), p(ln), n, max(lens),
                                    total, H, D, code, 0, stream) == 0
    empty = [i for i in range(n) if i not in full]
    assert torch.equal(out["s"][empty], a["s0"][empty]) and torch.equal(out["ds0"][empty], a["d_s"][empty])
    ref.check({**out, "s": out["s"][full], "ds0": out["ds0"][full]}, want, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_packed_calls_captured_and_at_once(dtype):
    """One long sequence among short ones, from a graph that is replayed on other values, and from two streams at once: the same bits."""
    import rwkv_ops_b200 as ro
    g = torch.Generator().manual_seed(39)
    lens, H = [5, 900, 1, 40, 7, 130, 3, 3, 60], 2
    cu = torch.tensor([0] + lens).cumsum(0)
    p = ro.PackedSequences(cu, "cuda")

    def inputs(seed):
        x = ref.inputs(1, int(cu[-1]), H, dtype=dtype, w="head", seed=seed)
        x["d_s"] = 0.1 * torch.randn(len(lens), H, 64, 64, generator=g)
        return [x[q].cuda() for q in ("r", "w", "k", "v", "d_o", "d_s")]

    def call(t):
        a = [y.detach().requires_grad_(True) for y in t[:4]]
        o, s = ro.linear_attention_varlen(*a, p)
        return [y.detach() for y in (o, s, *torch.autograd.grad((o, s), a, t[4:]))]

    one, two = inputs(40), inputs(41)
    want = [call(one), call(two)]
    held = [t.clone() for t in one]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(held)
    for i, src in ((1, two), (0, one)):
        for t, y in zip(held, src):
            t.copy_(y)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        both = []
        for s, t in zip(streams, (one, two)):
            with torch.cuda.stream(s):
                both.append(call(t))
        torch.cuda.synchronize()
        for a, b in zip(both, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
