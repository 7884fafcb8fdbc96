"""Memory that a call of the beam operators both reads and writes, or writes twice.  What is refused is refused on the host (CPU);
what is allowed equals the call on copies (GPU)."""
import ctypes as C

import pytest
import torch

from vae_conditional_sampling_amd import _lib
from vae_conditional_sampling_amd.sampling.beam import reorder_states
from vae_conditional_sampling_amd.sampling.utils import QuantisedHistory

EINVAL = -1


def strides(*v):
    return (C.c_int64 * 3)(*v)


def test_parents_inside_the_destination_are_refused_at_the_entry():
    """4 x 2 x 3 rows of 8 bytes: 192 bytes, parents of 48."""
    L = _lib.lib()
    lay = strides(48, 24, 8)
    base = 1 << 20
    for src in (base, base + 4096):                      # in place, and out of place
        for parents in (base, base + 48, base + 184, base - 40):
            assert L.cs_beam_reorder(src, base, 4, 2, 3, 3, 8, lay, lay, parents, None) == EINVAL
            assert b"parents" in L.cs_last_error()


def test_outputs_and_states_of_the_ring_are_apart_from_what_is_read():
    """A ring of 5 x 2 x 3 records of 16 bytes (480 bytes), rows of 7 float32."""
    L = _lib.lib()
    ring = 1 << 20
    c = _lib.cs_qcache(ring, 5, 2, 3, 7, 0, 64)
    far = 1 << 22

    def read(out, stride, slots=None, chains=None, N=2, J=3):
        return L.cs_qcache_read(C.byref(c), slots, 0, chains, N, J, out, 0, strides(*stride), None)

    lay = (42, 21, 7)
    for stride in ((42, 21, 6), (42, 21, 0), (42, 20, 7), (41, 21, 7), (0, 21, 7), (42, 7, 7), (7, 13, 42), (42, -21, 7)):
        assert read(far, stride) == EINVAL
        assert b"overlap" in L.cs_last_error() or b"negative" in L.cs_last_error()
    for out in (ring, ring + 476, ring - 332):           # (2 x 2 x 3 rows: 336 bytes)
        assert read(out, lay) == EINVAL and b"lies in" in L.cs_last_error()
    for at in (far, far + 332, far - 92):                # (2 x 2 x 3 indices: 96 bytes)
        assert read(far, lay, slots=at) == EINVAL and b"lies in" in L.cs_last_error()
        assert read(far, lay, slots=far + 4096, chains=at) == EINVAL and b"lies in" in L.cs_last_error()
    for X in (ring, ring + 476, ring - 332):
        assert L.cs_qcache_write(C.byref(c), X, 0, 2, strides(*lay), None, 0, None, None) == EINVAL
        assert b"ring" in L.cs_last_error()
    assert L.cs_qcache_write(C.byref(c), far, 0, 2, strides(42, -21, 7), None, 0, None, None) == EINVAL


@pytest.mark.gpu
def test_rows_of_an_output_that_overlap_are_refused():
    q = QuantisedHistory(4, (2, 3, 7), "int8")
    q.write(torch.randn(4, 2, 3, 7, device="cuda"), 0)
    slots = torch.zeros(2, 2, 3, dtype=torch.int64, device="cuda")
    wide = torch.zeros(200, device="cuda")
    for stride in ((42, 21, 3, 1), (21, 21, 7, 1), (1, 21, 7, 1)):
        with pytest.raises(_lib.CsError, match="overlap"):
            q.read(slots, out=wide.as_strided((2, 2, 3, 7), stride))
    with pytest.raises(_lib.CsError, match="overlap"):
        q.read_steps(0, 2, out=wide.as_strided((2, 2, 3, 7), (40, 21, 7, 1)))
    assert not wide.any()
    with pytest.raises(_lib.CsError, match="lies in"):
        q.read(slots, out=q.data.reshape(-1)[:84 * 4].view(torch.float32).reshape(2, 2, 3, 7))
    for stride in ((60, 30, 10, 1), (7, 14, 28, 1), (7, 14, 42, 1), (21, 42, 7, 1), (7, 42, 14, 1)):     # any order of the axes
        out = torch.zeros(200, device="cuda").as_strided((2, 2, 3, 7), stride)
        assert torch.equal(q.read(slots, out=out), q.read(slots))


@pytest.mark.gpu
@pytest.mark.parametrize("K", [2, 4, 6, 40])
@pytest.mark.parametrize("B,T", [(3, 5), (700, 40)])
def test_a_history_of_parents_follows_its_own_last_row(B, T, K):
    g = torch.Generator().manual_seed(K)
    past = torch.randint(0, K, (T, B, K), generator=g).cuda()
    b = torch.arange(B, device="cuda")[:, None]
    for row in (0, T // 2, T - 1):
        want = past[:, b, past[row]]
        own = past.clone()
        assert reorder_states(own, own[row], batch_dim=1, out=own) is own
        assert torch.equal(own, want)
        into = past.clone()                              # out of place, the parents in what is written
        reorder_states(past, into[row], batch_dim=1, out=into)
        assert torch.equal(into, want)
        rows = past.transpose(0, 1).contiguous()         # [B,T,K]: parents with a stride
        moved = rows.transpose(0, 1)
        reorder_states(moved, moved[row], batch_dim=1, out=moved)
        assert torch.equal(moved, want)
