"""The operators for linear attention with a decay for each head, and for beam search over recurrent states: what a program
that trains, prefills or decodes with them asks of this package, through the public entry points.

Every case is a plain dict; ``kind`` names the call:

==============  ======================================================================================
``prefill``     ``linear_attention`` without gradients, final state returned
``train``       ``linear_attention`` forward + backward, gradients of every input
``packed``      ``linear_attention_varlen`` forward + backward over sequences packed end to end
``step``        one token on a resident state (``LinearAttentionDecodeState.step``); with ``beams`` > 1 every
                sequence continues from the state of the beam it was selected from (``parents``)
``select``      the best continuations of every beam search over beams x vocabulary (``beam_select``)
``reorder``     the rows of a resident state follow the selected beams (``Rwkv7DecodeState.reorder``)
==============  ======================================================================================

One (batch, head), g_t = -exp(w_t), S a matrix [value][key]:

    S_t = exp(g_t) S_{t-1} + v_t k_t^T        o_t = S_t r_t

``w`` is one number per head (``[H]``) or per token and head (``[B, T, H]``), float32.

With ``own`` false the operators are computed in their plain form, chunks of 64 tokens in float32 (decay sums in float64).
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
BYTES = {"bf16": 2, "f32": 4, "f16": 2}
CHUNK = 64


def listed():
    return [
        # interactive generation: one sequence, one token of one layer; the call itself is all there is
        dict(name="step, one sequence", kind="step", groups=1, beams=1, H=32, D=64, dtype="bf16", state="f32", w="head"),
        # a decode server's full batch
        dict(name="step, batch of 256", kind="step", groups=256, beams=1, H=64, D=64, dtype="bf16", state="f32", w="token"),
        # beam search on states kept in bfloat16: every beam continues from the one it was selected from
        dict(name="step, beams", kind="step", groups=21, beams=5, H=40, D=64, dtype="bf16", state="bf16", w="token"),
        # one user's prompt, of whatever length it has
        dict(name="prefill, one prompt", kind="prefill", B=1, T=1000, H=32, D=64, dtype="bf16", w="head", with_state=False),
        # long documents that continue from a state
        dict(name="prefill, long documents", kind="prefill", B=4, T=16384, H=32, D=64, dtype="bf16", w="token",
             with_state=True),
        # a small model's micro-batch (fine-tuning on short texts)
        dict(name="train, small", kind="train", B=2, T=371, H=12, D=64, dtype="bf16", w="token", with_state=False),
        # pre-training at 2048 channels
        dict(name="train, 2048 channels", kind="train", B=8, T=4096, H=32, D=64, dtype="bf16", w="token", with_state=False),
        # documents of very different lengths packed into one batch, a learned decay for each head
        dict(name="train, packed", kind="packed", n_seq=8, max_len=4096, H=32, D=64, dtype="bf16", w="head"),
        # float32 tokens, for those who need float32-exact gradients
        dict(name="train, float32", kind="train", B=2, T=1024, H=16, D=64, dtype="f32", w="token", with_state=True),
        # one beam search, four beams, a vocabulary of 65536
        dict(name="select, four beams", kind="select", groups=1, beams=4, V=65536, dtype="bf16", eos=False),
        # a batch of beam searches, an odd vocabulary, float32 logits, some beams finished
        dict(name="select, batch of 64", kind="select", groups=64, beams=8, V=50277, dtype="f32", eos=True),
        # the states of one layer follow the beams
        dict(name="reorder", kind="reorder", groups=64, beams=4, H=32, state="f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random):
    kind = rng.choice(("step", "step", "prefill", "prefill", "train", "train", "train", "packed", "select", "select", "reorder"))
    w = rng.choice(("head", "token"))
    if kind in ("step", "reorder"):
        beams = rng.choice((1, 1, 2, 3, 4, 6, 8)) if kind == "step" else rng.randint(2, 16)
        groups = _log_int(rng, 1, max(1, 256 // beams))
        state = rng.choice(("f32", "bf16"))
        if kind == "reorder":
            return dict(kind=kind, groups=groups, beams=beams, H=rng.randint(8, 64), state=state)
        D = rng.choice((64, 64, 64, 128))
        return dict(kind=kind, groups=groups, beams=beams, H=rng.randint(8, 4096 // D), D=D,
                    dtype=rng.choice(("bf16", "bf16", "f16", "f32")), state=state, w=w)
    if kind == "select":
        beams, groups = rng.randint(1, 16), _log_int(rng, 1, 128)
        most = max(512, min(131072, 64 * 8 * 50277 // (groups * beams)))
        return dict(kind=kind, groups=groups, beams=beams, V=_log_int(rng, 512, most),
                    dtype=rng.choice(("bf16", "f16", "f32")), eos=rng.random() < 0.5)
    dtype = rng.choice(("bf16", "bf16", "bf16", "bf16", "f32", "f16"))
    D = rng.choice((64, 64, 64, 128)) if dtype == "bf16" else 64
    if kind == "packed":
        n, length = _log_int(rng, 2, 24), _log_int(rng, 32, 6000)
        H = rng.randint(8, 48)
        if dtype != "bf16" or D == 128:      # float32 arithmetic: fewer tokens
            H, length = min(H, 16), min(length, 1500)
        return dict(kind=kind, n_seq=n, max_len=length, H=H, D=D, dtype=dtype, w=w)
    B, T, H = _log_int(rng, 1, 16), _log_int(rng, 1, 8192), rng.randint(8, 64)
    if dtype != "bf16" or D == 128:
        B, H, T = min(B, 4), min(H, 32), min(T, 2048)
    T = min(T, max(1, 8 * 4096 * 32 // (B * H)))
    return dict(kind=kind, B=B, T=T, H=H, D=D, dtype=dtype, w=w, with_state=rng.random() < 0.5)


def _lengths(case):
    """Sequence lengths of a packed batch: uniform in [max_len / 16, max_len], one of them max_len."""
    rng = random.Random("%d sequences of %d" % (case["n_seq"], case["max_len"]))
    lens = [rng.randint(max(1, case["max_len"] // 16), case["max_len"]) for _ in range(case["n_seq"])]
    lens[rng.randrange(len(lens))] = case["max_len"]
    return lens


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _parents(case):
    """Which beam of its group each beam continues from: the better ones more often, and often themselves.  The same for
    every seed, so that what a reordering has to move is known."""
    rng = random.Random("%d searches of %d" % (case["groups"], case["beams"]))
    W = case["beams"]
    return [[j if rng.random() < 0.4 else min(rng.randrange(W), rng.randrange(W)) for j in range(W)]
            for _ in range(case["groups"])]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    kind = case["kind"]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    st = {"kind": kind, "own": own}
    if kind == "select":
        G, W, V = case["groups"], case["beams"], case["V"]
        st["logits"] = (2.5 * normal(G, W, V)).to(DTYPES[case["dtype"]])
        st["logits"][..., V // 7] = -math.inf      # a token that is never to be generated
        # beams in order of their scores, as the step before has left them
        st["scores"] = -(3 + torch.rand(G, W, generator=g, device="cuda")).cumsum(1)
        st["finished"], st["eos"] = None, None
        if case["eos"]:
            st["finished"] = torch.rand(G, W, generator=g, device="cuda") < 0.2
            st["eos"] = V // 3
        return st
    if kind == "reorder":
        G, W, H = case["groups"], case["beams"], case["H"]
        state = (0.1 * normal(G * W, H, 64, 64)).to(DTYPES[case["state"]])
        st["parents"] = torch.tensor(_parents(case), device="cuda")
        if own:
            from rwkv_ops_b200 import Rwkv7DecodeState
            st["decoder"] = Rwkv7DecodeState(G * W, H, state_dtype=DTYPES[case["state"]], initial_state=state)
        else:
            st["state"] = state
        return st

    H, D, dtype = case["H"], case["D"], DTYPES[case["dtype"]]
    if kind == "step":
        B, T = case["groups"] * case["beams"], 1
    elif kind == "packed":
        lens = _lengths(case)
        B, T = 1, sum(lens)
    else:
        B, T = case["B"], case["T"]
    # keys of about unit length, as a normalised projection leaves them
    st["r"], st["k"], st["v"] = normal(B, T, H, D).to(dtype), (normal(B, T, H, D) / math.sqrt(D)).to(dtype), normal(B, T, H, D).to(dtype)
    # decays from 0.7 to 0.999 per token
    st["w"] = -3 + normal(H) if case["w"] == "head" else -3 + normal(B, T, H)
    if kind == "step":
        state = (0.1 * normal(B, H, D, D)).to(DTYPES[case["state"]])
        st["parents"] = torch.tensor(_parents(case), device="cuda") if case["beams"] > 1 else None
        if own:
            from rwkv_ops_b200 import LinearAttentionDecodeState
            st["decoder"] = LinearAttentionDecodeState(B, H, head_size=D, state_dtype=DTYPES[case["state"]], initial_state=state)
        else:
            st["state"] = state
        return st
    n = B
    if kind == "packed":
        n = len(lens)
        if own:
            from rwkv_ops_b200 import PackedSequences
            st["sequences"] = PackedSequences(_offsets(lens), "cuda")      # made once for all the layers of a step
        else:
            st["place"], st["valid"] = _padded(lens)
    st["initial_state"] = 0.1 * normal(n, H, D, D) if case.get("with_state") else None
    if kind != "prefill":
        st["d_out"] = normal(B, T, H, D).to(dtype)
        st["d_state"] = 0.1 * normal(n, H, D, D)
    return st


def _padded(lens):
    """Where the tokens of a packed batch lie in a padded one, and which of its [n_seq, max_len] places they take."""
    valid = torch.arange(max(lens), device="cuda")[None] < torch.tensor(lens, device="cuda")[:, None]
    return valid.flatten().nonzero()[:, 0], valid


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(st):
    return _run_own(st) if st["own"] else _run_plain(st)


def _run_own(st):
    import rwkv_ops_b200 as ro

    kind = st["kind"]
    if kind == "select":
        return ro.beam_select(st["logits"], st["scores"], finished=st["finished"], eos=st["eos"])
    if kind == "reorder":
        st["decoder"].reorder(st["parents"])
        return st["decoder"].state
    if kind == "step":
        o = st["decoder"].step(st["r"], st["w"], st["k"], st["v"], parents=st["parents"])
        return o, st["decoder"].state
    if kind == "prefill":
        with torch.no_grad():
            return ro.linear_attention(st["r"], st["w"], st["k"], st["v"], initial_state=st["initial_state"])
    args = [st[n].detach().requires_grad_(True) for n in "rwkv"]
    s0 = st["initial_state"]
    if s0 is not None:
        s0 = s0.detach().requires_grad_(True)
    if kind == "packed":
        o, s = ro.linear_attention_varlen(*args, st["sequences"], initial_state=s0)
    else:
        o, s = ro.linear_attention(*args, initial_state=s0)
    wrt = args if s0 is None else args + [s0]
    return (o, s) + torch.autograd.grad((o, s), wrt, (st["d_out"], st["d_state"]))


def _run_plain(st):
    kind = st["kind"]
    if kind == "select":
        return _plain_select(st["logits"], st["scores"], st["finished"], st["eos"])
    if kind == "reorder":
        G, W = st["parents"].shape
        rows = (st["parents"] + W * torch.arange(G, device="cuda")[:, None]).flatten()
        st["state"] = st["state"][rows]
        return st["state"]
    if kind == "step":
        return _plain_step(st)
    if kind == "prefill":
        with torch.no_grad():
            o, s = _plain_attention(st["r"].float(), st["w"], st["k"].float(), st["v"].float(), st["initial_state"])
            return o.to(st["r"].dtype), s
    dtype = st["r"].dtype
    args = [st[n].detach().float().requires_grad_(True) for n in "rwkv"]
    s0 = st["initial_state"]
    if s0 is not None:
        s0 = s0.detach().requires_grad_(True)
    if kind == "packed":
        place, valid = st["place"], st["valid"]

        def pad(x):
            return x.new_zeros(valid.numel(), *x.shape[2:]).index_copy(0, place, x[0]).unflatten(0, valid.shape)

        r, w, k, v = args
        o, s = _plain_attention(pad(r), w if w.dim() == 1 else pad(w), pad(k), pad(v), s0, valid)
        o = o.flatten(0, 1)[place][None]
    else:
        o, s = _plain_attention(*args, s0)
    wrt = args if s0 is None else args + [s0]
    grads = torch.autograd.grad((o, s), wrt, (st["d_out"].float(), st["d_state"]))
    cast = [dtype, torch.float32, dtype, dtype, torch.float32]
    return (o.detach().to(dtype), s.detach()) + tuple(x.to(t) for x, t in zip(grads, cast))


def _plain_attention(r, w, k, v, s0, valid=None):
    """[B, T, H, D] in float32: products inside chunks of 64 tokens, and a product over the chunks for the states."""
    B, T, H, D = r.shape
    g = -torch.exp(w.double())
    g = g.expand(B, T, H)
    if valid is not None:
        g = torch.where(valid[..., None], g, 0)      # what follows a sequence leaves its state alone
    N = -(-T // CHUNK)
    pad = N * CHUNK - T

    def chunks(x):      # [B, T, H, ...] -> [B, H, N, 64, ...]
        x = torch.cat([x, x.new_zeros(B, pad, *x.shape[2:])], 1) if pad else x
        return x.unflatten(1, (N, CHUNK)).movedim(3, 1)

    r, k, v, g = chunks(r), chunks(k), chunks(v), chunks(g)
    L = g.cumsum(-1)
    total = L[..., -1]
    far = L[..., :, None] - L[..., None, :]
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=r.device).tril()
    decay = torch.exp(torch.where(lower, far, -math.inf)).float()
    a = (r @ k.transpose(-1, -2)) * decay
    # what each chunk adds to the state, and the decays between the end of one chunk and the start of another
    add = v.transpose(-1, -2) @ (k * torch.exp(total[..., None] - L).float()[..., None])
    upto = total.cumsum(-1)
    before = torch.cat([torch.zeros_like(upto[..., :1]), upto], -1)      # sums of the chunks before n = 0 .. N
    far = before[..., :, None] - upto[..., None, :]
    lower = torch.ones(N + 1, N, dtype=torch.bool, device=r.device).tril(-1)
    between = torch.exp(torch.where(lower, far, -math.inf)).float()
    states = (between @ add.flatten(-2)).unflatten(-1, (D, D))
    if s0 is not None:
        states = states + torch.exp(before).float()[..., None, None] * s0[:, :, None]
    o = a @ v + (r * torch.exp(L).float()[..., None]) @ states[:, :, :-1].transpose(-1, -2)
    return o.movedim(1, 3).flatten(1, 2)[:, :T], states[:, :, -1]


def _plain_step(st):
    S = st["state"].float()
    if st["parents"] is not None:
        G, W = st["parents"].shape
        S = S[(st["parents"] + W * torch.arange(G, device="cuda")[:, None]).flatten()]
    r, k, v = (st[n][:, 0].float() for n in "rkv")
    d = torch.exp(-torch.exp(st["w"] if st["w"].dim() == 1 else st["w"][:, 0]))
    S = S * d[..., None, None] + v[..., :, None] * k[..., None, :]
    o = (S * r[..., None, :]).sum(-1)
    st["state"] = S.to(st["state"].dtype)
    return o.to(st["r"].dtype)[:, None], st["state"]


def _plain_select(logits, scores, finished, eos):
    G, W, V = logits.shape
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    x = x - (top + (x - top).exp().sum(-1, keepdim=True).log()) + scores.double()[..., None]
    token = torch.arange(V, device=x.device)
    if finished is not None:      # a finished beam goes on with `eos` alone, at the score it has
        x = torch.where(finished[..., None], torch.where(token == eos, scores.double()[..., None], -math.inf), x)
    x = x.reshape(G, W * V)
    least = x.topk(W).values[:, -1:]
    above, equal = x > least, x == least
    chosen = above | (equal & (equal.cumsum(-1) <= W - above.sum(-1, keepdim=True)))      # of equal ones the first
    place = W * V - torch.where(chosen, W * V - torch.arange(W * V, device=x.device), 0).topk(W).values
    best, order = x.gather(1, place).sort(dim=1, descending=True, stable=True)
    place = place.gather(1, order)
    parents, tokens = place // V, place % V
    if eos is None:
        return best.float(), parents, tokens
    return best.float(), parents, tokens, finished.gather(1, parents) | (tokens == eos)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "select":
        n = case["groups"] * case["beams"]
        return {"bytes": n * (case["V"] * BYTES[case["dtype"]] + 24), "flops": 4 * n * case["V"]}
    if kind in ("step", "reorder"):
        G, W, H, D = case["groups"], case["beams"], case["H"], case.get("D", 64)
        state = H * D * D * BYTES[case["state"]]
        p = _parents(case) if W > 1 else [[0]] * G
        if kind == "reorder":      # beams that stay are neither read nor written
            read = sum(len({q for j, q in enumerate(x) if q != j}) for x in p)
            write = sum(sum(q != j for j, q in enumerate(x)) for x in p)
            return {"bytes": max(1, (read + write) * state) + 8 * G * W, "flops": 0}
        read = sum(len(set(x)) for x in p)
        w = H * 4 * (G * W if case["w"] == "token" else 1)
        return {"bytes": (read + G * W) * state + 4 * G * W * H * D * BYTES[case["dtype"]] + w, "flops": 5 * G * W * H * D * D}
    H, D = case["H"], case["D"]
    if kind == "packed":
        lens = _lengths(case)
        n, tokens = len(lens), sum(lens)
    else:
        n, tokens = case["B"], case["B"] * case["T"]
    one, state = tokens * H * D * BYTES[case["dtype"]], n * H * D * D * 4
    w = 4 * H * (tokens if case["w"] == "token" else 1)
    has = 1 if case.get("with_state") else 0
    if kind == "prefill":
        return {"bytes": 4 * one + w + (1 + has) * state, "flops": 4 * tokens * H * D * D}
    return {"bytes": 8 * one + 2 * w + (2 + 2 * has) * state, "flops": 14 * tokens * H * D * D}


# ---------------------------------------------------------------------------------------------
# the definition, token by token in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind == "reorder":
        return None
    was = own
    globals()["own"] = False
    try:
        st = prepare(case, seed)
    finally:
        globals()["own"] = was
    if kind == "select":
        return _exact_select(st)
    if kind == "step":
        S = st["state"].double()
        if st["parents"] is not None:
            S = S.unflatten(0, tuple(st["parents"].shape))
            S = torch.stack([x[p] for x, p in zip(S, st["parents"])]).flatten(0, 1)
        w = st["w"].double().expand(S.shape[0], 1, case["H"])
        S = torch.exp(-torch.exp(w[:, 0]))[..., None, None] * S + torch.einsum("bhv,bhk->bhvk", st["v"][:, 0].double(), st["k"][:, 0].double())
        return torch.einsum("bhvk,bhk->bhv", S, st["r"][:, 0].double())[:, None], S
    r, k, v = (st[n].double() for n in "rkv")
    w = st["w"].double()
    valid = st.get("valid")

    def pad(x):      # sequences of a packed batch side by side, zeros behind them
        if valid is None:
            return x
        y = x.new_zeros(*valid.shape, *x.shape[2:])
        y[valid] = x[0]
        return y

    def pack(x):
        return x if valid is None else x[valid][None]

    g = -torch.exp(w.expand(*r.shape[:3]))
    r, k, v, gp = pad(r), pad(k), pad(v), pad(g)
    n, T, H, D = r.shape
    d = torch.exp(gp)
    S = torch.zeros(n, H, D, D, dtype=torch.float64, device="cuda") if st["initial_state"] is None else st["initial_state"].double()
    o = torch.empty_like(r)
    if kind == "prefill":
        for t in range(T):
            S = torch.addcmul(d[:, t, :, None, None] * S, v[:, t, :, :, None], k[:, t, :, None, :])
            o[:, t] = (S @ r[:, t, :, :, None])[..., 0]
        return o, S
    do = pad(st["d_out"].double())
    dr, dk, dv, dg = (torch.empty_like(x) for x in (r, k, v, gp))
    for t in range(T):
        S = torch.addcmul(d[:, t, :, None, None] * S, v[:, t, :, :, None], k[:, t, :, None, :])
        o[:, t] = (S @ r[:, t, :, :, None])[..., 0]
        dr[:, t] = (do[:, t, :, None, :] @ S)[..., 0, :]
    last = S
    dS = st["d_state"].double()
    # dg_t = <dS_t, d_t S_{t-1}>, the product of state and gradient followed backwards over the tokens
    inner = (dS * S).sum((-1, -2))
    for t in reversed(range(T)):
        dS = torch.addcmul(dS, do[:, t, :, :, None], r[:, t, :, None, :])
        inner = inner + (do[:, t] * o[:, t]).sum(-1)                                   # <dS_t, S_t>
        dk[:, t] = (v[:, t, :, None, :] @ dS)[..., 0, :]
        dv[:, t] = (dS @ k[:, t, :, :, None])[..., 0]
        inner = inner - (dk[:, t] * k[:, t]).sum(-1)                                   # <dS_t, d_t S_{t-1}>
        dg[:, t] = inner
        dS = d[:, t, :, None, None] * dS
    dw = pack(dg) * g
    if st["w"].dim() == 1:
        dw = dw.sum((0, 1))
    out = (pack(o), last, pack(dr), dw, pack(dk), pack(dv))
    return out if st["initial_state"] is None else out + (dS,)


def _exact_select(st):
    import numpy as np

    x, s = st["logits"].double().cpu().numpy(), st["scores"].double().cpu().numpy()
    fin = None if st["finished"] is None else st["finished"].cpu().numpy()
    best = np.empty(s.shape)
    W = s.shape[1]
    for i in range(s.shape[0]):
        found = []
        for j in range(W):
            if fin is not None and fin[i, j]:
                found += [s[i, j]]
                continue
            row = np.partition(x[i, j], x.shape[2] - W)[-W:]
            top = row.max()
            found += list(s[i, j] + row - top - math.log(np.exp(x[i, j] - top).sum()))
        found += [-math.inf] * W
        best[i] = sorted(found, reverse=True)[:W]
    out = (best, None, None)
    return out if st["eos"] is None else out + (None,)
