"""Copies of a QuantisedHistory, and a ring that is put in the place of another (CPU: which memory the library is given; GPU:
what it does there)."""
import copy
import io
import pickle

import pytest
import torch

from vae_conditional_sampling_amd.sampling.utils import QuantisedHistory


def given(q):
    return q._desc.data


def test_a_copy_has_a_ring_of_its_own():
    q = QuantisedHistory(4, (2, 3, 7), "int8", group=32, device="cpu")
    q.data.random_(0, 256)
    own = q.data.data_ptr()
    shallow = copy.copy(q)
    assert shallow.data is q.data and given(shallow) == own
    shallow.data = q.data.clone()                        # (a snapshot: the original stays where it was)
    assert given(q) == own == q.data.data_ptr() and given(shallow) == shallow.data.data_ptr() != own
    for other in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert torch.equal(other.data, q.data) and given(other) == other.data.data_ptr() != own
        assert (other.fmt, other.group, other.record_bytes, other._desc.D) == ("int8", 32, q.record_bytes, 7)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "mxfp8", "mxfp4"])
def test_copies_are_written_and_read_apart(fmt):
    g = torch.Generator().manual_seed(1)
    q = QuantisedHistory(4, (2, 3, 43), fmt)
    q.write(torch.randn(4, 2, 3, 43, generator=g).cuda(), 0)
    before = q.read_steps(0, 4)
    other = copy.copy(q)
    other.data = q.data.clone()
    other.write(torch.randn(4, 2, 3, 43, generator=g).cuda(), 0)
    assert torch.equal(q.read_steps(0, 4), before) and not torch.equal(other.read_steps(0, 4), before)
    file = io.BytesIO()
    torch.save(q.data, file)
    file.seek(0)
    other.data = torch.load(file, weights_only=True)
    assert torch.equal(other.read_steps(0, 4), before)
