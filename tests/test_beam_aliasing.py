"""Memory that a call of the beam operators both reads and writes, or writes twice.  What is refused is refused on the host (CPU);
what is allowed equals the call on copies (GPU)."""
import ctypes as C

import pytest
import torch

from vae_conditional_sampling_amd import _lib
from vae_conditional_sampling_amd.sampling.beam import reorder_states

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
