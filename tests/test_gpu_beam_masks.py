"""Shapes of masks: what broadcasts to the logits and what is refused."""
import pytest
import torch

from vae_conditional_sampling_amd import _lib
from vae_conditional_sampling_amd.sampling.beam import beam_select

pytestmark = pytest.mark.gpu


def test_masks_that_do_not_broadcast_are_refused_like_other_arguments():
    logits = torch.randn(2, 3, 8, device="cuda")
    for shape in ((2, 3, 7), (2, 2, 8), (3, 3, 8), (2, 1), (1, 2, 3, 8), (2, 3, 0)):
        with pytest.raises(_lib.CsError, match="broadcast"):
            beam_select(None, logits, 2, mask=torch.ones(shape, dtype=torch.bool, device="cuda"))
    for shape in ((), (8,), (1,), (3, 1), (3, 8), (2, 1, 1), (1, 3, 8), (2, 3, 8)):
        got = beam_select(None, logits, 2, mask=torch.ones(shape, dtype=torch.bool, device="cuda"))
        assert all(torch.equal(a, b) for a, b in zip(got, beam_select(None, logits, 2)))
