"""The normaliser of the beam selection where sums are hard: a token that outweighs a long faint tail, logits that rise along the row, a row left to
one warp."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# (149 groups and more have one CTA of 16 warps each: with 16 beams a row is one warp's)
SIZES = [(1, 4, 50277), (1, 2, 65536), (40, 8, 50277), (150, 16, 131072)]


def rows(kind, W, V, seed):
    """[W, V] float32 logits that are bfloat16 numbers (differences of these are exact in float32 down to 2^-24 of the largest)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    noise = torch.randn(W, V, generator=g, device="cuda")
    if kind == "one token and a faint tail":
        x = torch.full((W, V), -16.75, device="cuda")
        x[:, 0] = 0.0
    elif kind == "one token last":
        x = torch.full((W, V), -11.0, device="cuda")
        x[:, -1] = 0.0
    elif kind == "rising":
        x = torch.linspace(-20, 2, V, device="cuda").expand(W, V) + 0.01 * noise
    elif kind == "falling":
        x = torch.linspace(2, -20, V, device="cuda").expand(W, V) + 0.01 * noise
    elif kind == "masks":      # most tokens forbidden, by the lowest number or by -inf
        x = torch.where(noise > 1.5, 2.5 * noise, torch.where(noise > 0, -torch.inf, torch.finfo(torch.bfloat16).min))
    else:
        x = 2.5 * noise
    return x.bfloat16()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["one token and a faint tail", "one token last", "rising", "falling", "masks", "mild"])
@pytest.mark.parametrize("G,W,V", SIZES)
def test_scores_of_hard_sums(G, W, V, kind, dtype):
    import rwkv_ops_b200 as ro
    distinct = rows(kind, 3, V, V + W)
    logits = distinct.to(dtype)[torch.arange(G * W, device="cuda") % 3].view(G, W, V)
    x = distinct.double()
    norm = torch.logsumexp(x, 1)[torch.arange(G * W, device="cuda") % 3].view(G, W)
    g = torch.Generator(device="cuda").manual_seed(G)
    scores = -(3 * torch.rand(G, W, generator=g, device="cuda")).cumsum(1)
    best, parents, tokens = ro.beam_select(logits, scores)
    row = (torch.arange(G, device="cuda")[:, None] * W + parents) % 3
    want = scores.double().gather(1, parents) + x[row, tokens] - norm.gather(1, parents)
    # A term of the sum is off by 2^-22 (the exponential), a tile's 16 are added in four roundings of 2^-24, a lane's sum is multiplied by two rounded factors
    # at most while it matters (2^-23 each, the product as much again) and by two more exponentials when lanes and warps meet (2^-23 each): 2^-20 in all; the
    # score is rounded once.
    off = (best.double() - want).abs() - 2.0 ** -24 * want.abs()
    assert float(off.max()) <= 2.0 ** -20, float(off.max())
    # and they are the best: the W-th of the exact scores of all candidates, a few groups at a time
    for s in range(0, G, 25):
        r = slice(s, min(G, s + 25))
        least = (scores[r].double()[..., None] + x[(torch.arange(r.start * W, r.stop * W, device="cuda") % 3)].view(-1, W, V)
                 - norm[r][..., None]).flatten(1).topk(W).values
        assert ((least - want[r]).abs() <= 2.0 ** -19).all()
