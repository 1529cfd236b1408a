"""Linear attention with a decay for each head against its definition in float64: lengths, types, layouts, decays, gradients,
packed batches, streams, graphs, and the recurrent form."""
import math

import pytest
import torch

import linear_attention_reference as ref

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def run(x, *, head_first=False, cu=None, device="cuda"):
    import rwkv_ops_b200 as ro

    def lay(t):
        return t.transpose(1, 2).contiguous() if head_first else t

    a = {n: (x[n] if x[n].dim() == 1 else lay(x[n])).to(device).requires_grad_(True) for n in "rwkv"}
    s0 = None if x["s0"] is None else x["s0"].to(device).requires_grad_(True)
    if cu is None:
        o, s = ro.linear_attention(*[a[n] for n in "rwkv"], initial_state=s0, head_first=head_first)
    else:
        o, s = ro.linear_attention_varlen(*[a[n] for n in "rwkv"], cu, initial_state=s0)
    assert o.dtype == x["r"].dtype and s.dtype == F32 and o.shape == a["r"].shape
    wrt = [a[n] for n in "rwkv"] + ([] if s0 is None else [s0])
    g = torch.autograd.grad((o, s), wrt, (lay(x["d_o"]).to(device), x["d_s"].to(device)))
    out = dict(zip(["o", "s", "dr", "dw", "dk", "dv", "ds0"], [o, s, *g]))
    return {n: lay(t) if n not in ("s", "ds0") and t.dim() > 2 else t for n, t in out.items()}


@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 64), (F16, 64), (F32, 128), (BF16, 128)])
@pytest.mark.parametrize("B,T,H,w,n_state", [(2, 1, 3, "token", 2), (1, 2, 1, "head", 0), (1, 63, 2, "token", 1), (2, 64, 2, "head", 1),
                                             (1, 65, 3, "token", 0), (1, 127, 1, "token", 1), (2, 128, 2, "token", 2),
                                             (1, 129, 2, "head", 1), (3, 200, 2, "token", 1), (1, 385, 5, "head", 0)])
def test_against_the_definition(dtype, D, B, T, H, w, n_state):
    x = ref.inputs(B, T, H, D, dtype=dtype, w=w, n_state=n_state, seed=T)
    ref.check(run(x), ref.with_gradients(x), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("w", ["token", "head"])
def test_head_first(dtype, w):
    x = ref.inputs(2, 150, 3, dtype=dtype, w=w, n_state=2, seed=5)
    want = ref.with_gradients(x)
    ref.check(run(x, head_first=True), want, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("w_mean,w_std", [(-8.0, 0.5), (0.0, 1.0), (1.5, 1.0), (3.0, 2.0)])
def test_slow_and_fast_decays(dtype, w_mean, w_std):
    """From states that hardly decay to ones that a token or two clear: exact in either case."""
    x = ref.inputs(1, 300, 2, dtype=dtype, n_state=1, w_mean=w_mean, w_std=w_std, seed=6)
    ref.check(run(x), ref.with_gradients(x), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padding_and_resets(dtype):
    """w = -1e9 leaves the state alone, w = +inf, the largest float32 and 100 clear it; gradients stay finite."""
    x = ref.inputs(2, 260, 2, dtype=dtype, n_state=2, seed=7)
    x["w"][0, 100:140] = -1e9
    x["w"][0, 3] = 100.0
    x["w"][1, 64] = math.inf
    x["w"][1, 130:136] = torch.finfo(F32).max
    x["w"][1, 200] = -math.inf
    x["w"][1, 201] = torch.finfo(F32).min
    y = dict(x)
    y["w"] = x["w"].clamp(-700, 6.5)      # (the definition's own gradient multiplies infinity by zero: e^{-e^{6.5}} is zero in float64 as well)
    ref.check(run(x), ref.with_gradients(y), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_infinity_stays_behind_a_reset_of_another_chunk(dtype):
    """What a token leaves cannot reach the tokens before its chunk."""
    import rwkv_ops_b200 as ro
    x = ref.inputs(1, 600, 2, dtype=dtype, seed=8)
    a = [x[n].cuda() for n in "rwkv"]
    o, _ = ro.linear_attention(*a)
    a[3][0, 520, 0, 3] = math.inf
    p, _ = ro.linear_attention(*a)
    assert torch.equal(o[:, :512], p[:, :512]) and torch.equal(o[:, :, 1], p[:, :, 1])
    assert not torch.isfinite(p[0, 520, 0, 3])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_decay_that_is_not_a_number_is_seen(dtype):
    import rwkv_ops_b200 as ro
    x = ref.inputs(1, 400, 2, dtype=dtype, seed=23)
    a = [x[n].cuda() for n in "rwkv"]
    o, _ = ro.linear_attention(*a)
    a[1][0, 300, 1] = math.nan
    p, s = ro.linear_attention(*a)
    assert torch.equal(o[:, :256], p[:, :256]) and torch.equal(o[:, :, 0], p[:, :, 0])
    assert torch.isnan(p[0, 301:, 1]).all() and torch.isnan(s[0, 1]).all()


@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 64), (F16, 128)])
@pytest.mark.parametrize("w,n_state", [("token", 4), ("head", 1)])
def test_packed(dtype, D, w, n_state):
    """Sequences end to end are what they are alone, and leave each other alone (NaN in one of them included)."""
    lens = [1, 130, 64, 257]
    cu = [0, 1, 131, 195, 452]
    T, H = cu[-1], 2
    x = ref.inputs(1, T, H, D, dtype=dtype, w=w, seed=9)
    g = torch.Generator().manual_seed(10)
    x["s0"], x["d_s"] = 0.1 * torch.randn(n_state, H, D, D, generator=g), 0.1 * torch.randn(4, H, D, D, generator=g)
    parts = []
    for i, n in enumerate(lens):
        y = {q: x[q][:, cu[i]:cu[i + 1]] if x[q].dim() == 4 or q == "w" and w == "token" else x[q] for q in ("r", "w", "k", "v", "d_o")}
        y["s0"] = x["s0"][i:i + 1] if n_state == 4 else x["s0"]
        y["d_s"] = x["d_s"][i:i + 1]
        parts.append(ref.with_gradients(y))
    want = {q: torch.cat([p[q] for p in parts], 1) for q in ("o", "dr", "dk", "dv")}
    want["s"] = torch.cat([p["s"] for p in parts])
    want["dw"] = sum(p["dw"] for p in parts) if w == "head" else torch.cat([p["dw"] for p in parts], 1)
    want["ds0"] = torch.cat([p["ds0"] for p in parts]) if n_state == 4 else sum(p["ds0"] for p in parts)
    got = run(x, cu=cu)
    # (the shared gradients of four sequences: sums of rows that are right each, of which one may be much larger)
    ref.check(got, want, dtype)
    bad = dict(x)
    bad["v"] = x["v"].clone()
    bad["v"][0, 131:195] = math.nan
    other = run(bad, cu=torch.tensor(cu))
    for q in ("o", "dr", "dk", "dv"):
        assert torch.equal(other[q][:, :131], got[q][:, :131]) and torch.equal(other[q][:, 195:], got[q][:, 195:]), q
    assert torch.isnan(other["o"][:, 131:195]).all()


@pytest.mark.parametrize("B,T,H,w,with_state", [
    (1, 2100, 1, "token", True),       # every chunk of 128 a part of its own, chained by a kernel
    (1, 1500, 1, "head", True),        # parts that put their start together themselves
    (9, 3000, 11, "token", False),     # two parts forward, the pass before them in finer pieces; one part backward
    (1, 5000, 24, "head", True),       # parts in both directions, the last chunk cut short
    (2, 1100, 37, "token", True),
])
def test_parts_of_few_sequences_are_the_whole(B, T, H, w, with_state):
    """Few sequences are walked in parts at once; bfloat16 tokens against the float32 operator, which has no parts, on the same values."""
    import rwkv_ops_b200 as ro
    g = torch.Generator(device="cuda").manual_seed(T)

    def n(*s):
        return torch.randn(*s, generator=g, device="cuda")

    x = [n(B, T, H, 64).bfloat16(), (-3 + n(H) if w == "head" else -3 + n(B, T, H)), (n(B, T, H, 64) / 8).bfloat16(), n(B, T, H, 64).bfloat16()]
    s0 = 0.1 * n(B, H, 64, 64) if with_state else None
    d_o, d_s = n(B, T, H, 64).bfloat16(), 0.1 * n(B, H, 64, 64)

    def call(dtype):
        a = [t if t.dtype == F32 else t.to(dtype) for t in x]
        a = [t.requires_grad_(True) for t in (u.detach().clone() for u in a)]
        s = None if s0 is None else s0.clone().requires_grad_(True)
        o, ht = ro.linear_attention(*a, initial_state=s)
        wrt = a if s is None else a + [s]
        return dict(zip(["o", "s", "dr", "dw", "dk", "dv", "ds0"], [o, ht, *torch.autograd.grad((o, ht), wrt, (d_o.to(dtype), d_s))]))

    ref.check(call(BF16), {q: t.detach().double().cpu() for q, t in call(F32).items()}, BF16)


def test_parts_of_packed_sequences():
    """Packed sequences of very different lengths, few enough to be walked in parts: short ones have none of the later parts."""
    import rwkv_ops_b200 as ro
    lens, H = [2500, 3, 700, 128, 1], 3
    cu = torch.tensor([0] + lens).cumsum(0)
    T = int(cu[-1])
    g = torch.Generator(device="cuda").manual_seed(22)

    def n(*s):
        return torch.randn(*s, generator=g, device="cuda")

    x = [n(1, T, H, 64).bfloat16(), -3 + n(1, T, H), (n(1, T, H, 64) / 8).bfloat16(), n(1, T, H, 64).bfloat16()]
    s0, d_o, d_s = 0.1 * n(5, H, 64, 64), n(1, T, H, 64).bfloat16(), 0.1 * n(5, H, 64, 64)
    x = [t.requires_grad_(True) for t in x]
    s0.requires_grad_(True)
    o, s = ro.linear_attention_varlen(*x, cu, initial_state=s0)
    packed = dict(zip(["o", "s", "dr", "dw", "dk", "dv", "ds0"], [o, s, *torch.autograd.grad((o, s), [*x, s0], (d_o, d_s))]))
    alone = []
    for i in range(5):
        cut = slice(int(cu[i]), int(cu[i + 1]))
        y = [t[:, cut].detach().to(BF16 if t.dim() == 4 else F32).float().requires_grad_(True) for t in x]
        z = s0[i:i + 1].detach().requires_grad_(True)
        o, s = ro.linear_attention(*y, initial_state=z)
        alone.append([o, s, *torch.autograd.grad((o, s), [*y, z], (d_o[:, cut].float(), d_s[i:i + 1]))])
    want = {q: torch.cat([a[j] for a in alone], 0 if q in ("s", "ds0") else 1).detach().double().cpu()
            for j, q in enumerate(["o", "s", "dr", "dw", "dk", "dv", "ds0"])}
    ref.check(packed, want, BF16)


def test_gradients_are_differences():
    """A directional derivative of a scalar of the outputs, against central differences of the float64 definition and of the operator itself."""
    import rwkv_ops_b200 as ro
    x = ref.inputs(1, 90, 2, n_state=1, seed=11)
    got = run(x)
    g = torch.Generator().manual_seed(12)
    for name, grad in (("r", "dr"), ("w", "dw"), ("k", "dk"), ("v", "dv"), ("s0", "ds0")):
        d = torch.randn(x[name].shape, generator=g)
        want = float((got[grad].double().cpu() * d.double()).sum())

        def value(e, f):
            y = {**x, name: x[name].double() + e * d}
            o, s = f(y)
            return float((o.double().cpu() * x["d_o"].double()).sum() + (s.double().cpu() * x["d_s"].double()).sum())

        e = 1e-4
        definition = lambda y: ref.linear_attention(y["r"], y["w"], y["k"], y["v"], y["s0"])
        diff = (value(e, definition) - value(-e, definition)) / (2 * e)
        scale = float(got[grad].double().norm() * d.double().norm()) / math.sqrt(d.numel())
        # curvature of the decays: e^2 times a third derivative that is of the size of the value
        assert abs(diff - want) <= 1e-4 * scale + 1e-6 * abs(diff), (name, diff, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_and_cast_inputs(dtype):
    """Views of a projection's output, w in the tokens' type, a state that is a view: as their contiguous copies."""
    import rwkv_ops_b200 as ro
    B, T, H, D = 2, 70, 3, 64
    g = torch.Generator().manual_seed(13)
    packed = torch.randn(B, T, 3, H, D, generator=g).to(dtype).cuda()
    r, k, v = packed.unbind(2)
    w = (-3 + torch.randn(B, T, H, generator=g)).to(BF16).cuda()
    s0 = torch.randn(B, H, D, D, generator=g).cuda().transpose(2, 3)
    o, s = ro.linear_attention(r, w, k, v, initial_state=s0)
    p, t = ro.linear_attention(r.contiguous(), w.float(), k.contiguous(), v.contiguous(), initial_state=s0.contiguous())
    assert torch.equal(o, p) and torch.equal(s, t)
    alone = ro.linear_attention(r, w, k, v, initial_state=s0, output_final_state=False)
    assert torch.equal(alone, o)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_results_twice_on_another_stream_and_from_a_graph(dtype):
    import rwkv_ops_b200 as ro
    x = ref.inputs(2, 333, 3, dtype=dtype, w="head", n_state=2, seed=14)
    first = run(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = run(x)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    for n in first:
        assert torch.equal(first[n], second[n]), n
    a = {n: x[n].cuda().requires_grad_(True) for n in ("r", "w", "k", "v", "s0")}
    d_o, d_s = x["d_o"].cuda(), x["d_s"].cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s = ro.linear_attention(a["r"], a["w"], a["k"], a["v"], initial_state=a["s0"])
        grads = torch.autograd.grad((o, s), list(a.values()), (d_o, d_s))
    with torch.no_grad():
        for t in a.values():
            t.mul_(0.5)
    graph.replay()
    with torch.no_grad():
        for t in a.values():
            t.mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    for n, t in zip(["o", "s", "dr", "dw", "dk", "dv", "ds0"], [o, s, *grads]):
        assert torch.equal(first[n], t), n


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_backward_without_kept_states(dtype, monkeypatch):
    x = ref.inputs(2, 210, 2, dtype=dtype, n_state=1, seed=15)
    kept = run(x)
    monkeypatch.setenv("RWKV_OPS_B200_KEEP_LIMIT_MB", "0")
    again = run(x)
    for n in kept:
        assert torch.equal(kept[n], again[n]), n


def test_gradients_of_one_output_alone_and_twice():
    import rwkv_ops_b200 as ro
    x = ref.inputs(1, 100, 2, dtype=BF16, n_state=1, seed=16)
    a = {n: x[n].cuda().requires_grad_(True) for n in ("r", "w", "k", "v", "s0")}
    o, s = ro.linear_attention(a["r"], a["w"], a["k"], a["v"], initial_state=a["s0"])
    d_o, d_s = x["d_o"].cuda(), x["d_s"].cuda()
    both = torch.autograd.grad((o, s), list(a.values()), (d_o, d_s), retain_graph=True)
    from_o = torch.autograd.grad(o, list(a.values()), d_o, retain_graph=True, allow_unused=True)
    again = torch.autograd.grad((o, s), list(a.values()), (d_o, d_s), retain_graph=True)
    zero = torch.autograd.grad((o, s), list(a.values()), (d_o, torch.zeros_like(d_s)))
    for p, q, u, z in zip(both, again, from_o, zero):
        assert torch.equal(p, q) and torch.equal(u, z)
    o2, _ = ro.linear_attention(a["r"], a["w"], a["k"], a["v"], initial_state=a["s0"])
    g, = torch.autograd.grad(o2.float().sum(), a["r"], create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


# ---------------------------------------------------------------------------------------------
# the recurrent form
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,state_dtype", [(F32, F32), (BF16, F32), (F16, BF16), (BF16, BF16)])
@pytest.mark.parametrize("w", ["token", "head"])
def test_steps_are_the_operator(D, dtype, state_dtype, w):
    import rwkv_ops_b200 as ro
    B, T, H = 3, 20, 2
    x = ref.inputs(B, T, H, D, dtype=dtype, w=w, n_state=1, seed=17)
    o, s = ref.linear_attention(*[x[n] for n in "rwkv"], initial_state=x["s0"])
    dec = ro.LinearAttentionDecodeState(B, H, head_size=D, state_dtype=state_dtype, initial_state=x["s0"].cuda())
    got = []
    for t in range(T):
        a = [x[n].cuda() if x[n].dim() == 1 else x[n][:, t:t + 1].cuda() for n in "rwkv"]
        if t % 2:
            a = [y if y.dim() == 1 else y[:, 0] for y in a]
        got.append(dec.step(*a).reshape(B, 1, H, D))
    got = torch.cat(got, 1).double().cpu()
    assert got.shape == o.shape
    # a rounding of the output; a bfloat16 state is rounded once a token, and the roundings of T tokens add up
    u = {F32: 2.0 ** -22, BF16: 2.0 ** -8, F16: 2.0 ** -11}
    tol = u[dtype] + (T * 2.0 ** -8 / 2 if state_dtype == BF16 else 2.0 ** -22)
    assert ((got - o).norm(dim=-1) / o.norm(dim=-1).clamp(min=float(o.norm(dim=-1).mean()))).max() <= tol
    tol = T * 2.0 ** -8 / 2 if state_dtype == BF16 else 2.0 ** -20
    assert float((dec.final_state().double().cpu() - s).norm() / s.norm()) <= tol


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_bfloat16_state_is_that_of_float32_arithmetic(dtype, D):
    """Bit for bit, over the steps of an answer (without a decay: its exponential is not the same everywhere)."""
    import rwkv_ops_b200 as ro
    B, T, H = 2, 12, 3
    x = ref.inputs(B, T, H, D, dtype=dtype, n_state=B, seed=24)
    dec = ro.LinearAttentionDecodeState(B, H, head_size=D, state_dtype=BF16, initial_state=x["s0"].cuda())
    S = x["s0"].to(BF16)
    none = torch.full((H,), -1e9)
    for t in range(T):
        r, k, v = (x[n][:, t].float() for n in "rkv")
        S = S.float() * 1.0 + v[..., :, None] * k[..., None, :]
        o = (S.double() * r[..., None, :].double()).sum(-1)
        size = (S.double() * r[..., None, :].double()).abs().sum(-1)
        S = S.to(BF16)
        got = dec.step(x["r"][:, t].cuda(), none.cuda(), x["k"][:, t].cuda(), x["v"][:, t].cuda())
        assert torch.equal(dec.state.cpu(), S), t
        # D products added in float32, at most D roundings of at most the sum of their sizes; and a rounding to the type
        off = (got.double().cpu() - o).abs() - torch.finfo(dtype).eps / 2 * o.abs()
        assert bool((off <= D * 2.0 ** -24 * size).all()), t


@pytest.mark.parametrize("state_dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("groups,beams", [(3, 1), (2, 2), (4, 3), (2, 5), (1, 8), (2, 11), (1, 32)])
def test_a_step_with_parents_is_a_reordering_and_a_step(groups, beams, D, state_dtype):
    import rwkv_ops_b200 as ro
    B, H = groups * beams, 3
    x = ref.inputs(B, 1, H, D, dtype=BF16, n_state=B, seed=18)
    a = [x[n].cuda() for n in "rwkv"]
    g = torch.Generator().manual_seed(19)
    parents = torch.randint(0, beams, (groups, beams), generator=g).cuda()
    one = ro.LinearAttentionDecodeState(B, H, head_size=D, state_dtype=state_dtype, initial_state=x["s0"].cuda())
    two = ro.LinearAttentionDecodeState(B, H, head_size=D, state_dtype=state_dtype, initial_state=x["s0"].cuda())
    rows = (parents + beams * torch.arange(groups, device="cuda")[:, None]).flatten()
    three = ro.LinearAttentionDecodeState(B, H, head_size=D, state_dtype=state_dtype, initial_state=x["s0"].cuda()[rows])
    o = one.step(*a, parents=parents)
    two.reorder(parents)
    assert torch.equal(two.state, three.state)
    p, q = two.step(*a), three.step(*a)
    assert torch.equal(o, p) and torch.equal(o, q)
    assert torch.equal(one.state, two.state) and torch.equal(one.state, three.state)
    # indices outside the search stay inside it; any whole numbers will do
    far = torch.where(parents == 0, -7, torch.where(parents == beams - 1, beams + 100, parents)) if beams > 1 else parents - 5
    four = ro.LinearAttentionDecodeState(B, H, head_size=D, state_dtype=state_dtype, initial_state=x["s0"].cuda())
    four.reorder(far.to(torch.int32))
    assert torch.equal(four.state, x["s0"].cuda()[rows].to(state_dtype))


@pytest.mark.parametrize("state_dtype", [F32, BF16])
def test_rwkv7_states_follow_beams(state_dtype):
    import rwkv_ops_b200 as ro
    G, W, H = 5, 6, 3
    g = torch.Generator().manual_seed(20)
    s = torch.randn(G * W, H, 64, 64, generator=g).to(state_dtype).cuda()
    parents = torch.randint(0, W, (G, W), generator=g).cuda()
    dec = ro.Rwkv7DecodeState(G * W, H, state_dtype=state_dtype, initial_state=s)
    version = dec.state._version
    dec.reorder(parents)
    assert torch.equal(dec.state, s[(parents + W * torch.arange(G, device="cuda")[:, None]).flatten()])
    assert dec.state._version > version
    small = torch.arange(4 * 3 * 8, dtype=torch.float16, device="cuda").view(12, 8)      # rows of 16 bytes, and a wider one with an odd count
    assert torch.equal(ro.reorder_states(small.clone(), torch.tensor([[2, 2, 0]] * 4, device="cuda")).view(4, 3, 8), small.view(4, 3, 8)[:, [2, 2, 0]])
    wide = torch.randn(4, 4 * 777, generator=g).cuda()
    assert torch.equal(ro.reorder_states(wide.clone(), torch.tensor([[1, 0, 3, 2]], device="cuda")), wide[[1, 0, 3, 2]])


def test_many_groups_and_large_states():
    import rwkv_ops_b200 as ro
    G = 70000      # more than a grid's second dimension
    s = torch.arange(2 * G * 4, dtype=F32, device="cuda").view(2 * G, 4)
    p = torch.tensor([1, 0], device="cuda").expand(G, 2)
    assert torch.equal(ro.reorder_states(s.clone(), p).view(G, 2, 4), s.view(G, 2, 4).flip(1))


def test_refusals():
    import rwkv_ops_b200 as ro
    x = ref.inputs(2, 8, 3, seed=21, n_state=2)
    r, w, k, v, s0 = (x[n].cuda() for n in ("r", "w", "k", "v", "s0"))
    for bad in ([r, w, k[:1], v], [r, w[:, :4], k, v], [r, w[0, 0, :2], k, v], [r[..., :32], w, k[..., :32], v[..., :32]],
                [r[0], w, k[0], v[0]], [r[:, :0], w[:, :0], k[:, :0], v[:, :0]], [r, w.T, k, v]):
        with pytest.raises(ValueError):
            ro.linear_attention(*bad)
    with pytest.raises(ValueError):
        ro.linear_attention(r, w, k, v, initial_state=s0[:, :2])
    with pytest.raises(ValueError):
        ro.linear_attention_varlen(r, w, k, v, [0, 8])
    for cu in ([0, 4], [0, 4, 4, 8], [1, 8], [0, 9]):
        with pytest.raises(ValueError):
            ro.linear_attention_varlen(r[:1], w[:1], k[:1], v[:1], cu)
    with pytest.raises(ro._lib.RwkvB200Error):
        ro.linear_attention(r, w.cpu(), k, v)
    dec = ro.LinearAttentionDecodeState(2, 3)
    one = [t[:, :1] for t in (r, w, k, v)]
    dec.step(*one)
    for parents in (torch.zeros(2, dtype=torch.long, device="cuda"), torch.zeros(3, 1, dtype=torch.long, device="cuda"),
                    torch.zeros(1, 2, device="cuda"), torch.zeros(2, 2, dtype=torch.long, device="cuda")):
        with pytest.raises(ValueError):
            dec.step(*one, parents=parents)
        with pytest.raises(ValueError):
            dec.reorder(parents)
    with pytest.raises(ro._lib.RwkvB200Error):
        dec.reorder(torch.zeros(1, 2, dtype=torch.long))
    with pytest.raises(ValueError):
        dec.step(r, w, k, v)
    with pytest.raises(ValueError):
        dec.step(one[0], w[:, :1, :2], one[2], one[3])
    with pytest.raises(ValueError):
        ro.LinearAttentionDecodeState(2, 3, state_dtype=F16)
    with pytest.raises(ValueError):
        ro.LinearAttentionDecodeState(2, 3, head_size=32)
    with pytest.raises(ValueError):
        ro.reorder_states(torch.zeros(66, 4, device="cuda"), torch.zeros(2, 33, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        ro.reorder_states(torch.zeros(4, 3, device="cuda"), torch.zeros(2, 2, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        ro.reorder_states(torch.zeros(4, 8, device="cuda")[:, ::2], torch.zeros(2, 2, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        ro.reorder_states(torch.zeros(4, 4, device="cuda", requires_grad=True), torch.zeros(2, 2, dtype=torch.long, device="cuda"))
