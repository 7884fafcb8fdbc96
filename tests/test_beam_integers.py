"""Integers that the C entries' types cannot hold are refused, not cut to some other value.  (CPU, and on the GPU shapes of
2^32 examples by a stride of zero: refused before anything is allocated.)"""
import pytest
import torch

from vae_conditional_sampling_amd import _lib
from vae_conditional_sampling_amd.sampling import beam
from vae_conditional_sampling_amd.sampling.utils import QuantisedHistory

FAR = (1 << 32) + 2          # cut to 32 bits: 2


def test_configurations():
    good = dict(B=2, K=3, V=10, width=4, logits_type=0, scores_type=0, normalise=1, end_token=0, ls0=30, ls1=10, ms0=0, ms1=0)
    assert beam._select_cfg(*good.values())[1] > 0
    for bad in (dict(B=FAR), dict(K=FAR), dict(end_token=FAR), dict(end_token=(1 << 64) + 1), dict(end_token=-1)):
        with pytest.raises(_lib.CsError):
            beam._select_cfg(*{**good, **bad}.values())


def test_layouts_and_rings():
    with pytest.raises(_lib.CsError, match="chains"):
        beam._rows((1, 2, FAR, 3), (0, 0, 0, 1), 4, 1)
    assert beam._rows((FAR, 2, 2, 3), (12, 6, 3, 1), 4, 1)[0] == FAR       # (64 bits for the other axes)
    assert beam._rows((2, FAR, 2, 3), (6 * FAR, 6, 3, 1), 4, 1)[3] == 4 * 12 * FAR
    for T, shape, group in ((FAR, (2, 3, 7), None), (4, (2, FAR, 7), None), (4, (2, 3, FAR), None), (4, (FAR, 3, 7), None),
                            (4, (2, 3, 7), (1 << 32) + 64)):
        with pytest.raises(_lib.CsError):
            QuantisedHistory(T, shape, "int8", group=group, device="meta")


def test_positions_and_steps():
    q = QuantisedHistory(7, (2, 3, 5), "int8", device="cpu")
    assert q._slot((1 << 64) + 5) == ((1 << 64) + 5) % 7 and q._slot(6) == 6 and q._slot(7) == 0
    assert q._slot(-1) < 0 and q._slot(-(1 << 64) + 3) < 0
    with pytest.raises(_lib.CsError, match="steps"):
        q.reorder(torch.zeros(2, 3, dtype=torch.int64), steps=-1)


@pytest.mark.gpu
def test_calls():
    one = torch.zeros(1, 1, 4, device="cuda")
    for shape in ((FAR, 1, 4), (1, FAR, 4)):
        with pytest.raises(_lib.CsError):
            beam.beam_select(None, one.expand(shape), 1)
    finished = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    for end in (FAR, (1 << 64) + 1, -1, 4):
        with pytest.raises(_lib.CsError, match="end token"):
            beam.beam_select(None, one, 1, finished=finished, end_token=end)
    q = QuantisedHistory(7, (1, 1, 5), "int8")
    x = torch.randn(1, 1, 5, device="cuda")
    q.write(x, (1 << 64) + 5)
    at = ((1 << 64) + 5) % 7
    assert q.read_steps(at, 1).abs().sum() > 0 and torch.equal(q.read_steps((1 << 70) + at - (1 << 70) % 7 + 7, 1), q.read_steps(at, 1))
    for start in (-1, -(1 << 64) + 1):
        with pytest.raises(_lib.CsError, match="start"):
            q.write(x, start)
        with pytest.raises(_lib.CsError, match="start"):
            q.read_steps(start, 1)
    with pytest.raises(_lib.CsError, match="slots"):
        q.read(torch.zeros(1, 1, dtype=torch.int64, device="cuda").expand(1, FAR), torch.zeros(1, 1, dtype=torch.int64, device="cuda").expand(1, FAR))
