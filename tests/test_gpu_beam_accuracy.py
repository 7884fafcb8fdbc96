"""Accuracy of the selection's 64-bit scores, against sums in 80 bits.

Bounds, derived: a term exp(x), |x| <= 40, is a table value (2^-53 relative), times a polynomial whose remainder is at most
(ln 2 / 128)^5 / 120 = 3.9e-14 and whose five steps round by 2^-53 each, of an argument that is off by at most |x| 2^-53 (the
rounding of ln 2 / 64, n times); 3.9e-14 + 46 * 1.1e-16 = 4.4e-14.  A lane adds 16 such terms, 6 steps join the lanes, and some 20 stretches
follow: 42 roundings, 5e-15.  The sum is divided by the largest term, itself off by 4.4e-14: in all 9.4e-14 relative, which is the absolute
error of its logarithm.  The score's own steps round four times, by 2^-53 of |x| + 2 |lse| + |score| at most."""
import numpy as np
import pytest
import torch

from vae_conditional_sampling_amd.sampling.beam import beam_select

pytestmark = pytest.mark.gpu


def lse80(x):
    x = np.asarray(x, dtype=np.longdouble)
    top = x.max(axis=-1, keepdims=True)
    return (top + np.log(np.exp(x - top).sum(axis=-1, keepdims=True)))[..., 0]


def compare(scores, logits, width, absolute):
    step = beam_select(scores.cuda(), logits.cuda(), width)
    got, parents, tokens = (t.cpu().numpy() for t in step)
    x = logits.double().numpy()
    lse = lse80(x)
    b = np.arange(x.shape[0])[:, None]
    x, lse, before = x[b, parents, tokens].astype(np.longdouble), lse[b, parents], scores.numpy().astype(np.longdouble)[b, parents]
    want = before + (x - lse)
    bound = absolute + 2.0 ** -53 * (np.abs(x) + 2 * np.abs(lse) + np.abs(want) + np.abs(before))
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,K,V,W", [(40, 3, 700, 8), (6, 2, 5000, 16), (2, 1, 40000, 5), (300, 4, 50, 4), (3000, 1, 2500, 3)])
def test_normalised_scores(dtype, B, K, V, W):
    g = torch.Generator().manual_seed(B)
    for scale, shift in ((1.0, 0.0), (4.0, 0.0), (0.05, 3.0), (3.0, -20.0)):
        logits = (torch.randn(B, K, V, generator=g) * scale + shift).to(dtype)
        compare(torch.randn(B, K, generator=g, dtype=torch.float64), logits, W, 9.4e-14)


@pytest.mark.parametrize("shift", [-5000.0, -650.0, 650.0, 5000.0])
def test_normalised_scores_relative_to_the_largest_logit(shift):
    """The sum is relative to that logit; differences are within 40, and float32's spacing at 5000 is 2^-11."""
    g = torch.Generator().manual_seed(9)
    logits = torch.randn(20, 2, 3000, generator=g) * 4 + shift
    compare(torch.randn(20, 2, generator=g, dtype=torch.float64), logits, 8, 9.4e-14)


@pytest.mark.parametrize("octave", [-1, 0, 1, 7])
def test_every_entry_of_the_table(octave):
    """999 equal terms 2^(octave - 1 + j / 64) beside one of 1 (or of 2^octave, where that is larger) for every j: the polynomial's
    argument is float32's rounding of the logit alone, so what is left is the table and the roundings, 46 + 42 of 1.1e-16 in the sum
    and 46 in what it is divided by: 1.5e-14."""
    top = max(octave, 0) * np.log(2.0)
    logits = torch.full((64, 1, 1000), 0.0, dtype=torch.float64)
    logits += ((octave - 1 + torch.arange(64, dtype=torch.float64) / 64) * np.log(2.0))[:, None, None]
    logits[:, :, 417] = top
    compare(torch.zeros(64, 1, dtype=torch.float64), logits.float(), 1, 1.5e-14)
