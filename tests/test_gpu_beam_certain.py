"""Beam selection where a beam's next token is certain: its total is the beam's score, to the bit, and ties go to the lowest beam."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


def _ops():
    from mindpipe_amd import ops
    return ops


def _certain(vocab, at, dtype, others):
    x = torch.full((vocab,), others, dtype=torch.float32)
    x[at] = 7.25
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab,at", [(1, 0), (300, 17), (32000, 31999), (128256, 70000)])
@pytest.mark.parametrize("others", [-INF, -2000.0])  # nothing else, or nothing that 64 bits see beside 1
def test_a_certain_token_keeps_its_score(dtype, vocab, at, others):
    """The logarithm of its share is 0.  Scores at 0 and near it, where a step of fp32 is far below what any sum is off by."""
    scores = [0.0, -1e-4, -1.0, -123.5, 0.5]
    x = torch.stack([_certain(vocab, at, dtype, others) for _ in scores]).to(DEV)
    have = torch.tensor([scores], device=DEV).t().contiguous()
    best, beam, token = _ops().beam_select(x, have, 1)
    assert torch.equal(best, have) and not beam.any() and (token == at).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 9000])
@pytest.mark.parametrize("score", [-1.0, 0.0, -1e-4])
def test_ended_and_certain_beams_tie(dtype, vocab, score):
    """An ended beam and one of the same score with one finite logit: the lowest beam first, both of the exact score."""
    x = torch.stack([_certain(vocab, 3, dtype, -INF)] * 2).to(DEV)
    have = torch.full((1, 2), score, device=DEV)
    for ended in ([True, False], [False, True]):
        best, beam, token = _ops().beam_select(x, have, 2, torch.tensor([ended], device=DEV), 1)
        assert torch.equal(best, have) and beam.tolist() == [[0, 1]]
        assert token.tolist() == [[1 if e else 3 for e in ended]]
        best, beam, token = _ops().beam_select(x, have, 1, torch.tensor([ended], device=DEV), 1)
        assert best.item() == have[0, 0].item() and beam.item() == 0


def test_a_step_of_the_score_decides():
    """Beams whose scores differ by one step of fp32, the lower one certain: it is not raised past the other."""
    x = torch.stack([_certain(400, 9, torch.float32, -INF)] * 2).to(DEV)
    for score in (-1e-4, -3e-6, -1e-9):
        high = torch.tensor(score, dtype=torch.float32)
        low = torch.nextafter(high, torch.tensor(-1.0))
        have = torch.stack((low, high))[None].to(DEV)
        best, beam, _ = _ops().beam_select(x, have, 2, torch.tensor([[False, True]], device=DEV), 1)
        assert beam.tolist() == [[1, 0]] and torch.equal(best, have.flip(1))


def test_shares_never_pass_one():
    """Scores of 0: no total is above it, whatever the others add.  Off by 2^-39 of what it is and 2^-45 (some hundred additions of
    fp64 to a sum near 1), and by half a step of fp32."""
    gaps = [700.0, 60.0, 36.0, 20.0, 12.0, 5.0, 1.0]
    x = torch.stack([torch.tensor([0.0, *[-g] * 63]) for g in gaps]).to(DEV)
    best = _ops().beam_select(x, torch.zeros(len(gaps), 1, device=DEV), 1)[0].flatten().tolist()
    for got, g in zip(best, gaps):
        want = -math.log1p(63 * math.exp(-g))
        assert got <= 0 and abs(got - want) <= (2.0 ** -24 + 2.0 ** -39) * abs(want) + 2.0 ** -45, g
