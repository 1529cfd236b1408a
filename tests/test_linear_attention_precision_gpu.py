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


@pytest.mark.parametrize("backward", [False, True])
def test_what_one_token_leaves_in_the_state(backward):
    """One token of 128 has a value (a gradient): the state is D v k^T (its gradient e^L d_o r^T), D the decay behind the token (L before and with it).  There is
    nothing to add up, so that only the factors and the parts of the scaled key (query) show: two exponentials of 2^-22, their product, that with
    the key and the rounded exponent 2^-24 each, and two sums of the three parts' products that cut off 2^-23 each: below 2^-20 of every element.
    Two parts instead of three leave up to 2^-17."""
    import rwkv_ops_b200 as ro
    B, T, H = 96, 128, 2
    x = ref.inputs(B, T, H, dtype=BF16, seed=42, w_mean=-8.0, w_std=0.3)
    at = torch.arange(B) * 4 // 3
    only = torch.zeros(B, T, 1, 1, dtype=torch.bool)
    only[torch.arange(B), at] = True
    g = -torch.exp(x["w"].double())
    rows = torch.arange(B)
    if backward:
        a = {q: x[q].cuda().requires_grad_(True) for q in "rwkv"}
        s0 = torch.zeros(B, H, 64, 64, device="cuda", requires_grad=True)
        o, s = ro.linear_attention(a["r"], a["w"], a["k"], a["v"], initial_state=s0)
        got, = torch.autograd.grad(o, s0, torch.where(only, x["d_o"], 0).cuda())
        D = torch.exp(g.cumsum(1))[rows, at]
        want = D[..., None, None] * x["d_o"].double()[rows, at, :, :, None] * x["r"].double()[rows, at, :, None, :]
    else:
        _, got = ro.linear_attention(x["r"].cuda(), x["w"].cuda(), x["k"].cuda(), torch.where(only, x["v"], 0).cuda())
        D = torch.exp(g.flip(1).cumsum(1).flip(1) - g)[rows, at]
        want = D[..., None, None] * x["v"].double()[rows, at, :, :, None] * x["k"].double()[rows, at, :, None, :]
    assert ((got.double().cpu() - want).abs() <= 2.0 ** -20 * want.abs()).all(), float(((got.double().cpu() - want) / want).abs().max())


def errors(got, want):
    """{name: the largest error of a row relative to its norm or the mean one} (a head's gradient of w is a row)."""
    out = {}
    for name, y in want.items():
        x = got[name].detach().double().cpu()
        if name == "dw":
            x, y = (x[None], y[None]) if y.dim() == 1 else (x.flatten(0, 1).T, y.flatten(0, 1).T)
        x, y = x.reshape(-1, x.shape[-1]), y.reshape(-1, y.shape[-1])
        norm = y.norm(dim=1)
        out[name] = float(((x - y).norm(dim=1) / norm.clamp(min=float(norm.square().mean().sqrt()))).max())
    return out


def run(x):
    import rwkv_ops_b200 as ro
    a = {n: x[n].cuda().requires_grad_(True) for n in ("r", "w", "k", "v", "s0")}
    o, s = ro.linear_attention(a["r"], a["w"], a["k"], a["v"], initial_state=a["s0"])
    return dict(zip(["o", "s", "dr", "dw", "dk", "dv", "ds0"], [o, s, *torch.autograd.grad((o, s), list(a.values()), (x["d_o"].cuda(), x["d_s"].cuda()))]))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("w,T", [("token", 300), ("head", 190)])
def test_float32_results(D, w, T):
    """A result of float32 tokens is some 3 D + T / 64 sums and ten factors in a chain, each rounded by 2^-24 at most of what has been summed: independent
    roundings add as their root, 400 of them and as much again for partial sums above the result 2^-19; in a row of D of them nothing cancels."""
    x = ref.inputs(2, T, 2, D, w=w, n_state=2, seed=43)
    for name, e in errors(run(x), ref.with_gradients(x)).items():
        assert e <= 2.0 ** -19, (name, e)


@pytest.mark.parametrize("w,T", [("token", 300), ("head", 700)])
def test_float32_results_of_bfloat16_tokens(w, T):
    """States and their gradients: three parts of the keys, 24 sums of a chunk that cut off up to 2^-23, and exponentials of 2^-22: 2^-18.  The gradient of w
    also takes products of states in two parts, 2^-17 of each element."""
    x = ref.inputs(2, T, 2, dtype=BF16, w=w, n_state=2, seed=44)
    got, want = run(x), ref.with_gradients(x)
    for name, e in errors(got, {n: want[n] for n in ("s", "ds0", "dw")}).items():
        assert e <= (2.0 ** -17 if name == "dw" else 2.0 ** -18), (name, e)


def test_gradients_are_differences_of_the_operator():
    """Central differences of the float32 operator itself.  It is linear in r, k, v and the first state, so that any step gives the derivative; in w the
    error of a step is a third of what changes with one of twice the size.  Results are good to 2^-19 of a row's norm (test_float32_results), which
    bounds what the differences and the sum over the gradient can be off by."""
    import rwkv_ops_b200 as ro
    x = ref.inputs(1, 90, 2, n_state=1, seed=45)
    got = run(x)
    g = torch.Generator().manual_seed(46)
    d_o, d_s = x["d_o"].double(), x["d_s"].double()
    for name in ("r", "w", "k", "v", "s0"):
        d = torch.randn(x[name].shape, generator=g)
        dot = float((got["d" + name].double().cpu() * d.double()).sum())

        def value(e):
            y = {**x, name: x[name] + e * d}
            o, s = ro.linear_attention(*[y[n].cuda() for n in "rwkv"], initial_state=y["s0"].cuda())
            o, s = o.double().cpu(), s.double().cpu()
            size = float((o.norm(dim=-1) * d_o.norm(dim=-1)).sum() + (s.norm(dim=-1) * d_s.norm(dim=-1)).sum())
            # (the argument is rounded, too: 2^-24 of it and of the outputs that it enters)
            return float((o * d_o).sum() + (s * d_s).sum()), size

        def difference(e):
            (p, a), (m, b) = value(e), value(-e)
            return (p - m) / (2 * e), (a + b) / (2 * e)

        e = 2.0 ** -6 if name == "w" else 1.0
        diff, size = difference(e)
        step = abs(difference(2 * e)[0] - diff) if name == "w" else 0.0
        rows = got["d" + name].double().cpu()
        flat = (lambda t: t.flatten(0, 1).T) if name == "w" else (lambda t: t.reshape(-1, t.shape[-1]))
        grad = float((flat(rows).norm(dim=1) * flat(d.double()).norm(dim=1)).sum())
        assert abs(diff - dot) <= 2.0 ** -19 * (size + grad) + step, (name, diff, dot)
        assert 2.0 ** -19 * (size + grad) + step <= 0.05 * grad, name      # (and that says something)


@pytest.mark.parametrize("backward", [False, True])
def test_sums_of_one_sign(backward):
    """Accumulators of tensor cores cut off instead of rounding, which adds up where all terms have one sign: over a chunk of 128 tokens the high part of the
    keys takes 8 steps of up to 2^-23 of sums that are half of the result on average, 2^-21, and the small parts, added before, next to nothing;
    two exponentials make as much again, 2^-20 in all.  (With the high part first the small ones cut off 16 times more: 1.6e-6 here.)"""
    import rwkv_ops_b200 as ro
    x = ref.inputs(2, 128, 2, dtype=BF16, seed=47, w_mean=-9.0, w_std=0.1)
    for q in ("r", "k", "v", "d_o"):
        x[q] = x[q].abs()
    x["s0"], x["d_s"] = torch.zeros(2, 2, 64, 64), torch.zeros(2, 2, 64, 64)
    name = "ds0" if backward else "s"
    got, want = run(x)[name].double().cpu(), ref.with_gradients(x)[name]
    assert ((got - want).abs() <= 2.0 ** -20 * want).all(), float(((got - want) / want).abs().max())


@pytest.mark.parametrize("side", ["first", "last"])
def test_gradients_of_decays_that_come_from_one_element(side):
    """One token reads one element of the first state (adds to one that a gradient of the last state meets): every decay between the two has a gradient of
    g D S[v][k], D the decay of all of them, and nothing is added up.  Three parts of the state are exact to 2^-24; two exponentials of 2^-22 and some six
    roundings of 2^-24 make less than 2^-20.  (Two parts leave up to 2^-17.)"""
    import rwkv_ops_b200 as ro
    B, T, H = 96, 128, 2
    x = ref.inputs(B, T, H, dtype=BF16, seed=48, w_mean=-7.0, w_std=0.3, n_state=B)
    gen = torch.Generator().manual_seed(49)
    at, vi, ki = torch.arange(B) * 4 // 3, torch.randint(0, 64, (B,), generator=gen), torch.randint(0, 64, (B,), generator=gen)
    n = torch.arange(B)
    key, value = torch.zeros(B, T, H, 64, dtype=BF16), torch.zeros(B, T, H, 64, dtype=BF16)
    key[n, at, :, ki], value[n, at, :, vi] = 1.0, 1.0
    zero, nothing = torch.zeros(B, T, H, 64, dtype=BF16), torch.zeros(B, H, 64, 64)
    g = -torch.exp(x["w"].double())
    t = torch.arange(T)[None]
    if side == "first":      # r, d_o and the first state
        r, k, v, d_o, s0, d_s, state = key, zero, zero, value, x["s0"], nothing, x["s0"]
        D, has = torch.exp(g.cumsum(1))[n, at], t <= at[:, None]
    else:
        r, k, v, d_o, s0, d_s, state = zero, key, value, zero, nothing, x["d_s"], x["d_s"]
        D, has = torch.exp(g.flip(1).cumsum(1).flip(1) - g)[n, at], t > at[:, None]
    w = x["w"].cuda().requires_grad_(True)
    o, s = ro.linear_attention(r.cuda(), w, k.cuda(), v.cuda(), initial_state=s0.cuda())
    got, = torch.autograd.grad((o, s), w, (d_o.cuda(), d_s.cuda()))
    want = torch.where(has[..., None], g * (D * state.double()[n, :, vi, ki])[:, None], 0)
    off = (got.double().cpu() - want).abs()
    assert (off <= 2.0 ** -20 * want.abs()).all(), float((off / want.abs().clamp(min=1e-30)).max())
