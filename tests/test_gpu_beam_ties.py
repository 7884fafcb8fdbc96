"""Scores that 64 bits do not tell apart although their logits differ: a beam's score far above the spacing of its logits, or
logits far below the spacing of their normaliser.  They go to the lowest (beam, value) like any equal scores.  Without a normaliser a score
is a sum of two given numbers, rounded once, so indices and scores are exact; with one, what is compared is the same whatever
its last bits are."""
import numpy as np
import pytest
import torch

from oracle import cs_oracle_beam as O
from vae_conditional_sampling_amd.sampling.beam import beam_select

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(scores, logits, width, *, exact=True, normalise=True, mask=None, finished=None, end_token=None):
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    step = beam_select(cuda(scores), cuda(logits), width, normalise=normalise, mask=cuda(mask), finished=cuda(finished), end_token=end_token)
    full = None if mask is None else np.broadcast_to(mask.numpy(), logits.shape)
    ref = O.beam_select(None if scores is None else scores.double().numpy(), logits.double().numpy(), width, normalise=normalise,
                        mask=full, finished=None if finished is None else finished.numpy(), end_token=end_token)
    assert np.array_equal(step.parents.cpu().numpy(), ref[1]), "parents"
    assert np.array_equal(step.tokens.cpu().numpy(), ref[2]), "tokens"
    if exact:
        want = torch.from_numpy(ref[0]).to(step.scores.dtype)
        assert torch.equal(step.scores.cpu(), want), "scores"
    return step


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [5, 40, 600, 3000, 20001])
def test_a_score_that_swallows_its_logits(dtype, V):
    g = torch.Generator().manual_seed(V)
    for W in (1, 4, 33, 64):
        for K in (1, 3):
            logits = (torch.randn(2, K, V, generator=g) * 3).to(dtype)
            for far in (-1e20, -3.4e38, 3e30, float("inf")):
                scores = torch.full((2, K), far, dtype=torch.float64)
                check(scores, logits, W)                       # tokens 0, 1, 2, ... of the first beam
                check(scores.float(), logits, W, normalise=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [8, 700, 5000])
def test_dead_beams_fill_the_places_behind_the_live_ones(dtype, V):
    g = torch.Generator().manual_seed(V + 1)
    B, K = 3, 4
    logits = (torch.randn(B, K, V, generator=g) * 2).to(dtype)
    mask = torch.ones(B, K, V, dtype=torch.bool)
    mask[:, 2] = torch.rand(B, V, generator=g) < 3 / V         # the live beam: a few continuations
    mask[:, 2, V // 2] = True
    mask[0, 0, :V // 4] = False
    for dead in (float(torch.finfo(torch.float32).min), -1e25):
        scores = torch.full((B, K), dead)
        scores[:, 2] = -1.5
        finished = torch.zeros(B, K, dtype=torch.bool)
        finished[1, 1] = True
        for W in (6, 16, 64):
            check(scores, logits, W, mask=mask, exact=False)
            check(scores, logits, W, mask=mask, normalise=False, finished=finished, end_token=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,W", [(1, 1, 300, 5), (2, 1, 2048, 5), (3, 1, 6000, 20), (2, 4, 3000, 16), (1, 16, 20000, 16), (2, 2, 9000, 64),
                                     (2, 64, 3000, 64), (1, 200, 70, 64), (2, 40, 500, 33), (700, 2, 500, 7), (300, 1, 10200, 5)])
def test_logits_in_classes_of_equal_scores(dtype, B, K, V, W):
    """2^57 and more: scores are multiples of 32, a class holds many logits of which any may come first."""
    g = torch.Generator().manual_seed(B + K + V + W)
    for scale in (8.0, 40.0, 400.0):
        logits = (torch.randn(B, K, V, generator=g) * scale).to(dtype)
        scores = torch.full((B, K), 1.5 * 2.0 ** 57, dtype=torch.float64)
        check(scores, logits, W, normalise=False)
        check(scores.float(), logits, W, normalise=False)
        scores += 32.0 * torch.randint(-3, 4, (B, K), generator=g)
        mask = torch.rand(B, 1, V, generator=g) < 0.5
        check(scores, logits, W, normalise=False, mask=mask)


@pytest.mark.parametrize("V", [300, 2048, 2049, 7000, 40000])
def test_logits_far_below_their_normaliser(V):
    """1e-20 beside a normaliser of log V or beside a score of one."""
    g = torch.Generator().manual_seed(V)
    for W in (1, 6, 40):
        logits = torch.randn(2, 1, V, generator=g) * 1e-20
        check(None, logits, W, exact=False)
        logits[0, 0, V // 2:] += 1.0                             # a class of ones ahead of it (the spacing there is 2^-23)
        logits[1, 0, V - 3:] = 2.0
        check(None, logits, W, exact=False)
        check(None, logits.bfloat16(), W, exact=False)
        two = logits.repeat(1, 2, 1)
        check(torch.tensor([[1.0, 1.0], [1.0, 3.0]]), two, W, normalise=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [400, 2048, 5000, 30000])
def test_equal_logits_beside_others_of_equal_score(dtype, V):
    """Zeros by the hundred, of which a stretch keeps the first W, and far ones that are larger but not in 64 bits, or smaller."""
    tiny = float(torch.finfo(dtype).tiny)
    for sign in (1.0, -1.0):
        for at in (slice(V - 20, V, 2), slice(V // 2, V // 2 + 90), slice(3, None, 7), slice(0, 30)):
            for W in (2, 16, 40, 64):
                logits = torch.zeros(1, 2, V, dtype=dtype)
                logits[0, 1, at] = sign * tiny
                scores = torch.tensor([[1000.0, 1000.0]])     # (float16's smallest normal, 2^-14, counts beside 1000)
                check(scores, logits, W, normalise=False)
                check(scores * 2.0 ** 40, logits, W, normalise=False)
                check(scores.double() * 2.0 ** 40, logits, W, exact=False)
                check(scores.flip(1) - torch.tensor([[0.0, 500.0]]), logits, W, normalise=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_rising_and_falling_logits_of_equal_score(dtype):
    for V in (500, 3000, 9000):
        rising = torch.arange(V, dtype=torch.float32).div(64).to(dtype)
        for row in (rising, rising.flip(0)):
            logits = row.repeat(2, 2, 1)
            scores = torch.tensor([[2.0 ** 56, 2.0 ** 56], [2.0 ** 56, 2.0 ** 56 + 64]], dtype=torch.float64)
            for W in (1, 12, 48, 64):
                check(scores, logits, W, normalise=False)


def test_an_example_does_not_depend_on_the_batch():
    """Stretches have 512, 1024 or 2048 values by the size of the call; what they keep differs, the result does not."""
    g = torch.Generator().manual_seed(8)
    V, W = 6000, 5
    logits = torch.randn(4096, 1, V, generator=g).bfloat16().cuda() * 8
    scores = torch.full((4096, 1), 2.0 ** 57, dtype=torch.float64, device="cuda")
    scores[::2] = -1e20
    whole = beam_select(scores, logits, W)
    for n in (1, 40, 400):
        part = beam_select(scores[:n], logits[:n], W)
        assert all(torch.equal(a, b[:n]) for a, b in zip(part, whole))
    assert torch.equal(whole.tokens[::2].cpu(), torch.arange(W).expand(2048, W))
