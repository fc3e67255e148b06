"""The order of beam selection's candidates whose scores are alike though their logits are not: beams without a score, and scores so
large that 64 bits no longer tell the logits apart."""
import pytest
import torch

from nemicli_terminal_b200 import beams

from tests.test_gpu_beams import BF16, F16, F32, define, gen

pytestmark = pytest.mark.gpu


def want(logits, scores, n):
    """Places k vocab + v of a request's n best: beams with a finite score by (score, beam, logit, place), all others and logits of -inf
    behind them by place.  For scores so far apart that no candidate of one beam comes near another's."""
    out = []
    for x, s in zip(logits.double().tolist(), scores.double().tolist()):
        vocab = len(x[0])
        live = [k for k in range(len(s)) if s[k] > -float("inf")]
        order = [(k, v) for k in sorted(live, key=lambda k: (-s[k], k)) for v in sorted(range(vocab), key=lambda v: (-x[k][v], v)) if x[k][v] > -float("inf")]
        order += sorted((k, v) for k in range(len(s)) for v in range(vocab) if k not in live or x[k][v] == -float("inf"))
        out.append([k * vocab + v for k, v in order[:n]])
    return out


def places(got, vocab):
    return (got[1].long() * vocab + got[2]).tolist()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dead", [float("-inf"), float("nan")])
@pytest.mark.parametrize("reqs, k, vocab, n", [(1, 1, 3, 3), (2, 3, 5, 15), (1, 4, 20001, 8), (3, 2, 131, 64), (40, 3, 9000, 33)])
def test_beams_without_a_score(cuda, dtype, dead, reqs, k, vocab, n):
    """Their candidates are all -inf: the lowest places, whatever the logits say, in every batch."""
    x = (torch.randn(reqs, k, vocab, generator=gen(vocab, cuda), device=cuda) * 3).to(dtype)
    x[:, -1, 1::2] = -float("inf")
    s = torch.full((reqs, k), dead, device=cuda)
    got = beams.select(x, s, n)                                   # all of them
    assert places(got, vocab) == [list(range(n))] * reqs and (got[0] == -float("inf")).all()
    s[:, -1] = -1.5                                               # the first ones, the last alive (every other token of it -inf)
    got = beams.select(x, s, n)
    assert places(got, vocab) == want(x, s, n)
    finite = min(n, (vocab + 1) // 2)
    assert torch.isfinite(got[0][:, :finite]).all() and (got[0][:, finite:] == -float("inf")).all()


def test_few_candidates_alive(cuda):
    """Fewer finite candidates than asked for, behind a beam without a score and before one."""
    x = torch.randn(1, 3, 40, generator=gen(1, cuda), device=cuda)
    x[0, 1, 5:] = -float("inf")
    s = torch.tensor([[-float("inf"), 0.5, -float("inf")]], device=cuda)
    got = beams.select(x, s, 60)
    assert places(got, 40) == want(x, s, 60)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("score", [-1e30, 3e25, float("inf")])
def test_scores_that_swallow_the_logits(cuda, dtype, score):
    """A score beside which fp64 holds no logit: the beam's candidates are still in the order of its logits, equal ones of their places."""
    x = (torch.randn(2, 2, 6007, generator=gen(6, cuda), device=cuda) * 2).to(dtype)
    s = torch.tensor([[score, -float("inf")], [-float("inf"), score]], device=cuda)
    got = beams.select(x, s, 40)
    assert places(got, 6007) == want(x, s, 40)


def test_logits_nearer_than_their_score_tells(cuda):
    """Logits of 1e-20 and 2e-20 under a largest one of 5: the scores are one number in fp64, the logits are not."""
    x = torch.full((1, 2, 3000), -9.0, device=cuda)
    x[0, :, 100] = 5.0
    x[0, :, 200:210] = torch.arange(10, device=cuda) * 1e-20
    s = torch.tensor([[0.0, -30.0]], device=cuda)
    got = beams.select(x, s, 8)
    assert places(got, 3000) == want(x, s, 8)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [9000, 140001])
def test_one_request_in_other_batches(cuda, dtype, vocab):
    """Rows are cut by how many there are, so a request's sums may differ in their last bits from batch to batch: by no more than the errors
    of two sums, and candidates further apart than that keep their places."""
    x = (torch.randn(80, 4, vocab, generator=gen(vocab, cuda), device=cuda) * 3).to(dtype)
    s = -torch.rand(80, 4, generator=gen(2, cuda), device=cuda).cumsum(1)
    exact, off = define(x[:2], s[:2])                             # (2, 4 vocab), (2, 1)
    best = torch.sort(exact, dim=1, descending=True)[0][:, :9]
    gap = torch.minimum((best[:, :-1] - best[:, 1:]), torch.nn.functional.pad(best[:, :-2] - best[:, 1:-1], (1, 0), value=float("inf")))
    clear = gap > 4 * off
    sizes = (2, 3, 20, 80)
    got = [[y[:2] for y in beams.select(x[:n], s[:n], 8)] for n in sizes]
    for n, here in zip(sizes, got):
        # twice the error of a sum, and the rounding of each score to float32
        assert ((here[0].double() - got[0][0].double()).abs() <= 2 * off + best[:, :8].abs() * 2.0 ** -23).all()
        assert all((a == b)[clear].all() for a, b in zip(here[1:], got[0][1:]))
        assert all(torch.equal(a[:2], b) for a, b in zip(beams.select(x[:n], s[:n], 8), here))      # the same batch: the same bits
