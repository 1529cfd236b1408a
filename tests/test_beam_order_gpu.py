"""The order of candidates whose scores differ by less than a float64 sum can tell: of one beam, the larger logit first, as in the choice of each beam's
own best; of two beams, the lower one."""
import pytest
import torch

import linear_attention_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("W", [1, 2, 3, 8, 32])
@pytest.mark.parametrize("rising", [False, True])
def test_logits_closer_than_a_sum_can_tell(W, rising):
    """Logits 1e-30 apart are different numbers, and the same score in float64."""
    import rwkv_ops_b200 as ro
    V = 700
    x = torch.arange(V) if rising else torch.arange(V).flip(0)
    logits = (1e-30 * x.float()).expand(2, W, V).contiguous()
    logits[1] *= -1
    scores = torch.zeros(2, W)
    scores[:, 1:] = -1e3      # one beam has all of the best
    got = ro.beam_select(logits.cuda(), scores.cuda())
    want = ref.beam_select(logits, scores)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2]), (got[2], want[2])
    eos = 5
    done = ro.beam_select(logits.cuda(), scores.cuda(), finished=torch.zeros(2, W, dtype=torch.bool, device="cuda"), eos=eos)
    assert torch.equal(done[2].cpu(), want[2]) and torch.equal(done[3].cpu(), want[2] == eos)


def test_equal_scores_of_two_beams_go_to_the_lower_one():
    import rwkv_ops_b200 as ro
    logits = torch.zeros(1, 2, 64)
    logits[0, 0, 40], logits[0, 1, 3] = 1e-30, 2e-30
    best, parents, tokens = ro.beam_select(logits.cuda(), torch.zeros(1, 2, device="cuda"))
    # (no score in float64 tells any of these 128 candidates from another: the lower beam, and there the larger logit, then the lower token)
    assert parents.tolist() == [[0, 0]] and tokens.tolist() == [[40, 0]] and float(best[0, 0]) == float(best[0, 1])
