"""Beam selection against its definition in float64, and a whole beam search over recurrent states against one that follows every
hypothesis from its first token."""
import math

import pytest
import torch

import linear_attention_reference as ref

pytestmark = pytest.mark.gpu


def check(logits, scores, finished=None, eos=None, move=lambda t: t):
    import rwkv_ops_b200 as ro
    got = ro.beam_select(move(logits.cuda()), scores.cuda(), finished=None if finished is None else finished.cuda(), eos=eos)
    want = ref.beam_select(logits, scores, finished, eos)
    assert len(got) == len(want)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int64
    assert torch.equal(got[1].cpu(), want[1]), (got[1], want[1], got[0], want[0])
    assert torch.equal(got[2].cpu(), want[2])
    # the sum under the logarithm: a few hundred float32 terms to a lane, each to within three roundings (2^-22); the score rounded once
    x, y = got[0].double().cpu(), want[0]
    assert torch.equal(torch.isfinite(x), torch.isfinite(y)) and torch.equal(x[~torch.isfinite(x)], y[~torch.isfinite(y)])
    fine = torch.isfinite(y)
    assert ((x - y)[fine].abs() <= 2.0 ** -21 + 2.0 ** -24 * y[fine].abs()).all()
    if eos is not None:
        assert torch.equal(got[3].cpu(), want[3])


def inputs(G, W, V, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(G, W, V, generator=g)).to(dtype), -(3 * torch.rand(G, W, generator=g)).cumsum(1), g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,W,V", [(1, 1, 1), (2, 1, 7), (1, 2, 1), (3, 4, 3), (1, 4, 1000), (2, 5, 4097), (4, 8, 2049), (1, 16, 777), (2, 32, 515),
                                   (1, 3, 20001), (300, 2, 33), (1, 32, 20)])
def test_against_the_definition(G, W, V, dtype):
    logits, scores, g = inputs(G, W, V, dtype, V + W)
    check(logits, scores)
    if V > 1:
        check(logits, scores, torch.rand(G, W, generator=g) < 0.4, V // 2)
        check(logits, scores, None, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("W", [1, 4, 32])
def test_ties_go_to_the_lowest(dtype, W):
    """Equal logits everywhere, few different ones, and beams that are copies of each other."""
    V = 3001
    scores = torch.zeros(2, W)
    check(torch.zeros(2, W, V, dtype=dtype), scores)
    g = torch.Generator().manual_seed(1)
    few = torch.randint(0, 3, (2, 1, V), generator=g).to(dtype).expand(2, W, V).contiguous()
    check(few, scores)
    rising = torch.arange(V).div(100, rounding_mode="floor").to(dtype).expand(2, W, V).contiguous()
    check(rising, scores)
    check(rising.flip(-1).contiguous(), scores)
    signs = torch.randint(0, 2, (2, 1, V), generator=g).expand(2, W, V).contiguous()
    check(torch.where(signs == 0, 0.0, -0.0).to(dtype), scores)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masked_tokens_dead_beams_and_bad_numbers(dtype):
    G, W, V = 2, 4, 600
    logits, scores, g = inputs(G, W, V, dtype, 3)
    logits[:, :, ::2] = -math.inf
    logits[0, 1] = -math.inf                     # a beam that cannot go on
    logits[0, 2, 5:] = torch.finfo(dtype).min    # masks of the type's lowest value
    logits[1, 0] = math.nan
    logits[1, 1, 17] = math.nan
    logits[1, 2, 9] = math.inf                   # an overflow, twice
    logits[1, 2, 100] = math.inf
    scores[1, 3] = -math.inf                     # a beam that does not exist yet
    check(logits, scores)
    check(logits, scores, torch.tensor([[True, False, False, True], [False, True, False, True]]), 599)
    first = torch.full((G, W), -math.inf)
    first[:, 0] = 0.0                            # the first step of a search: one beam
    check(inputs(G, W, V, dtype, 4)[0], first)
    nothing = torch.full((1, 3, 50), -math.inf, dtype=dtype)
    check(nothing, torch.zeros(1, 3))
    check(nothing, torch.full((1, 3), -math.inf), torch.tensor([[True, True, False]]), 7)
    check(nothing, torch.tensor([[math.nan, -1.0, -2.0]]), torch.tensor([[True, False, True]]), 0)


@pytest.mark.parametrize("W,V", [(4, 600), (3, 2), (32, 5), (32, 4000)])
def test_dead_beams(W, V):
    """Beams that do not exist (score -inf) go on with nothing: their candidates come last, the first tokens first, whatever their logits."""
    logits, scores, g = inputs(3, W, V, torch.float32, 9)
    scores[0] = -math.inf
    scores[1, 1:] = -math.inf
    scores[2, 0] = -math.inf
    logits[2, 1, 1:] = -math.inf
    check(logits, scores)
    check(logits, scores, torch.rand(3, W, generator=g) < 0.5, V - 1)


@pytest.mark.parametrize("eos", [0, 3, 31, 32, 40])
def test_all_beams_finished(eos):
    G, W, V = 2, 32, 41
    logits, scores, g = inputs(G, W, V, torch.float32, 5)
    scores[1, 7:] = -math.inf
    check(logits, scores, torch.ones(G, W, dtype=torch.bool), eos)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_strides_and_alignment(dtype, offset):
    """Rows cut out of a padded vocabulary, groups and beams in another order, a tensor that starts at an odd element."""
    G, W, V = 3, 4, 901
    logits, scores, g = inputs(G, W, V, dtype, 6)
    def padded(t):
        full = torch.full((W, G, V + 11), 1000.0, dtype=dtype, device="cuda")
        full[:, :, offset:offset + V] = t.transpose(0, 1)
        return full[:, :, offset:offset + V].transpose(0, 1)
    check(logits, scores, move=padded)
    check(logits, scores, move=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))      # (copied: the vocabulary is not the last in memory)
    shared = logits[:, :1].expand(G, W, V)
    check(shared.contiguous(), scores, move=lambda t: t[:, :1].expand(G, W, V))


def test_same_from_a_graph_and_on_another_stream():
    import rwkv_ops_b200 as ro
    logits, scores, g = inputs(2, 4, 5000, torch.bfloat16, 7)
    x, s = logits.cuda(), scores.cuda()
    want = ro.beam_select(x, s, eos=5)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = ro.beam_select(x, s, eos=5)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ro.beam_select(x, s, eos=5)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, other, got):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals():
    import rwkv_ops_b200 as ro
    x, s = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    f = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    for bad in (lambda: ro.beam_select(x[0], s), lambda: ro.beam_select(x, s[:1]), lambda: ro.beam_select(x[..., :0], s),
                lambda: ro.beam_select(x, s, finished=f), lambda: ro.beam_select(x, s, eos=50), lambda: ro.beam_select(x, s, eos=-1),
                lambda: ro.beam_select(x, s, finished=f[:1], eos=3),
                lambda: ro.beam_select(torch.zeros(1, 33, 5, device="cuda"), torch.zeros(1, 33, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ro._lib.RwkvB200Error):
        ro.beam_select(x.cpu(), s.cpu())
    with pytest.raises(ro._lib.RwkvB200Error):
        ro.beam_select(x, s.cpu())


@pytest.mark.parametrize("fused", [False, True])
def test_a_beam_search_over_recurrent_states(fused):
    """Prompt, then selections and steps on resident states; every hypothesis that is left has the score, and its state the value, that running
    its tokens through the operator from the start gives."""
    import rwkv_ops_b200 as ro
    G, W, H, V, T, steps = 2, 4, 2, 97, 70, 12
    g = torch.Generator().manual_seed(8)

    def n(*s):
        return torch.randn(*s, generator=g)

    emb = {q: n(V, H, 64).cuda() for q in "rkv"}
    emb["k"] = emb["k"] / 8
    w = (-2 + n(V, H)).cuda()
    head = (n(V, H * 64) / 4).cuda()
    prompt = torch.randint(0, V, (G, T), generator=g).cuda()

    def layer(tok):
        return emb["r"][tok], w[tok], emb["k"][tok], emb["v"][tok]

    o, s = ro.linear_attention(*layer(prompt))
    logits = (o[:, -1].flatten(1) @ head.T)[:, None].expand(G, W, V)
    dec = ro.LinearAttentionDecodeState(G * W, H, initial_state=s.repeat_interleave(W, 0))
    scores = torch.full((G, W), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    history = torch.empty(G, W, 0, dtype=torch.long, device="cuda")
    for _ in range(steps):
        scores, parents, tokens = ro.beam_select(logits, scores)
        history = torch.cat([history.gather(1, parents[..., None].expand(G, W, history.shape[2])), tokens[..., None]], 2)
        x = layer(tokens.flatten())
        if fused:
            o = dec.step(*x, parents=parents)
        else:
            dec.reorder(parents)
            o = dec.step(*x)
        logits = (o.flatten(1) @ head.T).view(G, W, V)
    full = torch.cat([prompt[:, None].expand(G, W, T), history], 2).flatten(0, 1)
    o64, s64 = ref.linear_attention(*[t.cpu() for t in layer(full)])
    lp = (o64.flatten(2) @ head.cpu().double().T).log_softmax(-1)
    want = lp[:, T - 1:-1].gather(2, full.cpu()[:, T:, None]).sum((1, 2)).view(G, W)
    assert len({tuple(h.tolist()) for h in history[0]}) == W
    # float32 products of 128 channels over the vocabulary, twelve times
    assert ((scores.double().cpu() - want).abs() <= 1e-3).all()
    assert (scores.diff(dim=1) <= 0).all()
    assert float((dec.final_state().double().cpu() - s64).norm() / s64.norm()) <= 2.0 ** -18
