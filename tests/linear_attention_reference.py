"""Linear attention with a decay for each head, token by token in float64 on the CPU, differentiable; and beam selection in plain Python."""
import math
from fractions import Fraction

import torch


def linear_attention(r, w, k, v, initial_state=None):
    """r, k, v [B, T, H, D], w [H] or [B, T, H]: o [B, T, H, D], final state [B, H, V, K], all float64."""
    r, w, k, v = (x.double() for x in (r, w, k, v))
    B, T, H, D = r.shape
    d = torch.exp(-torch.exp(w)).expand(B, T, H)
    S = torch.zeros(B, H, D, D, dtype=torch.float64) if initial_state is None else initial_state.double().expand(B, H, D, D)
    out = []
    for t in range(T):
        S = d[:, t, :, None, None] * S + v[:, t, :, :, None] * k[:, t, :, None, :]
        out.append((S * r[:, t, :, None, :]).sum(-1))
    return torch.stack(out, 1), S


def inputs(B, T, H, D=64, *, dtype=torch.float32, w="token", seed=0, n_state=0, w_mean=-3.0, w_std=1.0):
    """r, v ~ N(0, 1), k ~ N(0, 1 / D), w ~ N(w_mean, w_std^2) float32, states and their gradients ~ N(0, 0.1^2); rounded to `dtype`."""
    g = torch.Generator().manual_seed(seed)

    def n(*s):
        return torch.randn(*s, generator=g)

    x = {"r": n(B, T, H, D).to(dtype), "k": (n(B, T, H, D) / math.sqrt(D)).to(dtype), "v": n(B, T, H, D).to(dtype),
         "w": w_mean + w_std * (n(H) if w == "head" else n(B, T, H))}
    x["s0"] = 0.1 * n(n_state, H, D, D) if n_state else None
    x["d_o"], x["d_s"] = n(B, T, H, D).to(dtype), 0.1 * n(B, H, D, D)
    return x


def with_gradients(x):
    """What the operator and its backward return for inputs(): {name: float64 tensor}."""
    a = {n: x[n].double().requires_grad_(True) for n in "rwkv"}
    s0 = None if x["s0"] is None else x["s0"].double().requires_grad_(True)
    o, s = linear_attention(*[a[n] for n in "rwkv"], initial_state=s0)
    wrt = [a[n] for n in "rwkv"] + ([] if s0 is None else [s0])
    g = torch.autograd.grad((o, s), wrt, (x["d_o"].double(), x["d_s"].double()))
    return dict(zip(["o", "s", "dr", "dw", "dk", "dv", "ds0"], [o.detach(), s.detach(), *g]))


def tolerance(name, dtype):
    """Largest error of a row relative to its norm (or the mean one).

    Outputs in the tokens' type are rounded once (half a step u: 2^-8 bfloat16, 2^-11 float16), and where tensor cores are used the attention
    matrix is rounded to the type as well before its product: 2 u, and as much again for the sums of absolute values being larger than the
    sums.  float32 results (states, gradients of w, float32 tokens) come from products of exact or doubly split operands (2^-17 each, two of
    them) accumulated in float32: 2^-16, and as much again for the same reason.
    """
    if name in ("s", "dw", "ds0") or dtype == torch.float32:
        return 2.0 ** -15
    return 4 * torch.finfo(dtype).eps / 2


def check(got, want, dtype):
    """Every row of every tensor, against its norm or the mean norm of the rows, whichever is more."""
    for name, y in want.items():
        x = got[name].detach().double().cpu()
        assert x.shape == y.shape, (name, x.shape, y.shape)
        assert torch.isfinite(x).all(), name
        if name == "dw":      # a number per token and head: one row per head
            x, y = (x[None], y[None]) if y.dim() == 1 else (x.flatten(0, 1).T, y.flatten(0, 1).T)
        x, y = x.reshape(-1, x.shape[-1]), y.reshape(-1, y.shape[-1])
        norm = y.norm(dim=1)
        err = ((x - y).norm(dim=1) / norm.clamp(min=float(norm.square().mean().sqrt()) or 1.0)).max()
        assert err <= tolerance(name, dtype), (name, float(err), tolerance(name, dtype))


def beam_select(logits, scores, finished=None, eos=None):
    """The definition, candidate by candidate: the normaliser in float64, scores compared as the exact sums (a float64 sum would tie
    candidates of a row whose largest logit is the largest float32)."""
    G, W, V = logits.shape
    out = []

    def score(s, x, top, norm):
        return -math.inf if x == -math.inf or s == -math.inf else Fraction(s) + Fraction(x) - Fraction(top) - Fraction(norm)

    for g in range(G):
        found = []
        for i in range(W):
            s = float(scores[g, i])
            s = -math.inf if math.isnan(s) else s
            if finished is not None and finished[g, i]:
                found += [(s if t == eos else -math.inf, i, t) for t in range(V)]
                continue
            x = logits[g, i].double()
            x = torch.where(x < math.inf, x, -math.inf)      # (NaN too)
            top = x.max()
            if top == -math.inf:
                found += [(-math.inf, i, t) for t in range(V)]
            else:
                top, norm = float(top), float(torch.exp(x - top).sum().log())
                found += [(score(s, c, top, norm), i, t) for t, c in enumerate(x.tolist())]
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        out.append(found[:W])
    best = torch.tensor([[float(c[0]) for c in row] for row in out], dtype=torch.float64)
    parents = torch.tensor([[c[1] for c in row] for row in out])
    tokens = torch.tensor([[c[2] for c in row] for row in out])
    if eos is None:
        return best, parents, tokens
    was = torch.zeros(G, W, dtype=torch.bool) if finished is None else finished.cpu()
    return best, parents, tokens, was.gather(1, parents) | (tokens == eos)
