"""Copies of a QuantisedHistory, and a ring that is put in the place of another (CPU: which memory the library is given; GPU:
what it does there)."""
import copy
import io
import pickle

import pytest
import torch

from vae_conditional_sampling_amd.sampling.utils import ImputationHistoryQueue, QuantisedHistory


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


@pytest.mark.parametrize("storage", [None, "mxfp4"])
def test_a_queue_uses_the_ring_it_is_given(storage):
    q = ImputationHistoryQueue(4, (2, 3, 7), device="cpu", storage=storage)
    ring = q.history_queue.clone()
    q.history_queue = ring
    assert q.history_queue is ring
    if storage:
        assert given(q.quantised) == ring.data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("storage", [None, "int8", "mxfp8", "mxfp4"])
def test_a_queue_goes_on_with_a_restored_ring(storage):
    g = torch.Generator().manual_seed(2)
    X = [torch.randn(2, 3, 43, generator=g).cuda() for _ in range(4)]
    q, other = (ImputationHistoryQueue(4, (2, 3, 43), storage=storage) for _ in range(2))
    for x in X[:3]:
        q.enqueue_batch(x)
    other.history_queue, other.tail_idx, other.full = q.history_queue.clone(), q.tail_idx, q.full
    for queue in (q, other):
        queue.enqueue_batch(X[3])
    a, b = (queue.concat_history(X[0], [0, 2, 3], chain_of_proposal=[1, 0, 2]) for queue in (q, other))
    assert torch.equal(a, b) and bool(a[:, 3:].any())


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
