"""Beam search over chains: the deterministic sibling of the multinomial / systematic resampling.

The beams of an example are its chains ``[B,K]``; every beam can continue with ``V`` values (proposals, categories, tokens).
``beam_select`` keeps the ``width`` best continuations of an example, ``reorder_states`` lets what is kept per chain (latents
``[B,K,Zd]``, a history ``[T,B,K,D]``, drawn values) follow the chosen parents.  ``sampling.utils.QuantisedHistory`` keeps a
history in 8 or 4 bits and reorders it likewise.  The reference has no counterpart.
"""
import ctypes as C
import functools
from typing import NamedTuple, Optional

import torch

from .. import _lib

MAX_WIDTH = 64


class BeamStep(NamedTuple):
    scores: torch.Tensor    # [B,W], the type of the given scores
    parents: torch.Tensor   # [B,W] int64: the beam that is continued
    tokens: torch.Tensor    # [B,W] int64: the value it continues with


def _flags(t, what):
    """uint8 view of a bool / uint8 tensor."""
    if t.dtype == torch.bool:
        return t.view(torch.uint8)
    if t.dtype != torch.uint8:
        raise _lib.CsError(f"{what} must be a bool or uint8 tensor, got {t.dtype}")
    return t


@functools.lru_cache(maxsize=256)
def _select_cfg(B, K, V, width, logits_type, scores_type, normalise, end_token, ls0, ls1, ms0, ms1):
    """(cs_beam_cfg, bytes of workspace) of calls of one shape; read only."""
    if max(B, K, V, end_token) > _lib.INT32_MAX or end_token < 0:   # (they would wrap)
        raise _lib.CsError(f"at most 2^31 - 1 examples, beams and values and an end token among these, got {B}, {K}, {V}, {end_token}")
    pair = C.c_int64 * 2
    cfg = _lib.cs_beam_cfg(B, K, V, width, logits_type, scores_type, normalise, end_token, pair(ls0, ls1), pair(ms0, ms1))
    nbytes = _lib.lib().cs_beam_select_workspace(C.byref(cfg))
    if nbytes < 0:
        raise _lib.CsError(f"libcsvae error: {_lib.lib().cs_last_error().decode()}")
    return cfg, nbytes


def beam_select(scores: Optional[torch.Tensor], logits: torch.Tensor, width: int, *, normalise: bool = True,
                mask: Optional[torch.Tensor] = None, finished: Optional[torch.Tensor] = None,
                end_token: Optional[int] = None) -> BeamStep:
    """The ``width`` (1 .. 64) best continuations of every example, best first.

    ``scores`` [B,K] float32 / float64 (None: zeros, float32): what the beams have so far; -inf: a beam that is not in use (the
    first step of a search starts from one beam).  ``logits`` [B,K,V] float32 / bfloat16 / float16, the values adjacent in
    memory, any strides of the other axes.  A continuation scores
    ``scores + (logits - logsumexp(logits))``, or ``scores + logits`` with ``normalise=False``, formed in 64 bits;
    equal scores go to the lowest (beam, value), also where 64 bits do not tell different logits apart (a beam at -1e30).
    ``mask`` (bool, broadcastable to [B,K,V]; True = allowed): what is not allowed takes no part in the normaliser either and
    may hold anything.  ``finished`` [B,K] (bool): such a beam only continues with ``end_token``, at its score; its logits are
    not read.  NaN and -inf are never chosen; a beam with a NaN or +inf among its allowed logits has no continuations
    (``normalise``).  An example with fewer than ``width`` continuations ends in score -inf, token -1 and the slot's own index
    as parent."""
    if logits.dim() != 3:
        raise _lib.CsError(f"logits must be [B,K,V], got {tuple(logits.shape)}")
    B, K, V = logits.shape
    dev = _lib.on_device(logits, scores, mask, finished)
    logits_type = _lib.CS_TYPE.get(logits.dtype, 3)
    if logits_type == 3:
        raise _lib.CsError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    out_type, scores_at, mask_at, finished_at = torch.float32, None, None, None
    if scores is not None:
        out_type = scores.dtype
        if out_type not in (torch.float32, torch.float64):
            raise _lib.CsError(f"scores must be float32 or float64, got {out_type}")
        if scores.shape != (B, K):
            raise _lib.CsError(f"scores must be [{B},{K}], got {tuple(scores.shape)}")
        scores = scores.contiguous()
        scores_at = scores.data_ptr()
    ls = logits.stride()
    if ls[2] != 1 and V > 1:
        logits = logits.contiguous()
        ls = logits.stride()
    ms = (0, 0)
    if mask is not None:
        mask = _flags(mask, "mask")
        if mask.dim() > 3 or any(n not in (1, m) for n, m in zip(reversed(mask.shape), (V, K, B))):
            raise _lib.CsError(f"mask must broadcast to [{B},{K},{V}], got {list(mask.shape)}")
        mask = mask.expand(B, K, V)
        if mask.stride(2) != 1 and V > 1:
            mask = mask.contiguous()
        ms = mask.stride()
        mask_at = mask.data_ptr()
    if finished is None:
        end_token = 0
    else:
        if end_token is None:
            raise _lib.CsError("finished needs end_token")
        finished = _flags(finished, "finished")
        if finished.shape != (B, K):
            raise _lib.CsError(f"finished must be [{B},{K}], got {tuple(finished.shape)}")
        finished = finished.contiguous()
        finished_at = finished.data_ptr()
    width = int(width)
    if not 1 <= width <= MAX_WIDTH:
        raise _lib.CsError(f"width must be 1 .. {MAX_WIDTH}, got {width}")
    cfg, nbytes = _select_cfg(B, K, V, width, logits_type, _lib.CS_TYPE[out_type], int(bool(normalise)), int(end_token), ls[0],
                              ls[1], ms[0], ms[1])
    # the workspace is the call's own (calls on several streams and captured ones share nothing)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    new_scores = torch.empty((B, width), dtype=out_type, device=dev)
    parents = torch.empty((B, width), dtype=torch.int64, device=dev)
    tokens = torch.empty_like(parents)
    _lib.call_on(dev, _lib.lib().cs_beam_select, C.byref(cfg), scores_at, logits.data_ptr(), mask_at, finished_at,
                 new_scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(), work.data_ptr(), nbytes)
    return BeamStep(new_scores, parents, tokens)


@functools.lru_cache(maxsize=256)
def _rows(shape, strides, size, axis):
    """(outer, strides in bytes of (outer, example, chain), bytes of a row, bytes from the first row's start to the last one's
    end) of a tensor [outer..., B, K, row...], or None if the outer axes do not collapse into one stride or a row is not
    adjacent in memory."""
    if shape[axis + 1] > _lib.INT32_MAX:
        raise _lib.CsError(f"at most 2^31 - 1 chains, got {shape[axis + 1]}")
    row = 1
    for n, s in zip(reversed(shape[axis + 2:]), reversed(strides[axis + 2:])):
        if n != 1 and s != row:
            return None
        row *= n
    outer, stride = 1, 0
    for n, s in zip(reversed(shape[:axis]), reversed(strides[:axis])):
        if n == 1:
            continue
        if outer == 1:
            stride = s
        elif s != stride * outer:
            return None
        outer *= n
    end = (outer - 1) * stride + (shape[axis] - 1) * strides[axis] + (shape[axis + 1] - 1) * strides[axis + 1] + row
    return outer, (C.c_int64 * 3)(stride * size, strides[axis] * size, strides[axis + 1] * size), row * size, end * size


def reorder_states(states: torch.Tensor, parents: torch.Tensor, *, batch_dim: int = 0,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[..., b, w, ...] = states[..., b, parents[b, w], ...]`` for states of any type whose axes ``batch_dim`` and
    ``batch_dim + 1`` are examples and chains: latents [B,K,Zd], a history [T,B,K,D] (``batch_dim=1``).

    ``parents`` [B,W] int64; a parent outside [0,K) leaves its row of ``out`` as it was.  ``out=None`` returns a new tensor (a
    row without a parent is zero there: all of it is filled first, half as many bytes again); ``out=states`` works in place (W = K <= 64): rows that keep their place are not
    touched, so a search that leaves survivors where they are moves only what changed.  ``out`` elsewhere must not overlap
    ``states``.  ``parents`` may be a part of ``out`` (a history of parents that is reordered itself): it is copied first."""
    if batch_dim < 0:
        batch_dim += states.dim()
    if not 0 <= batch_dim <= states.dim() - 2:
        raise _lib.CsError("states need an example and a chain axis")
    shape = tuple(states.shape)
    B, K = shape[batch_dim:batch_dim + 2]
    if parents.dim() != 2 or parents.shape[0] != B or parents.dtype != torch.int64:
        raise _lib.CsError(f"parents must be int64 [{B},W], got {parents.dtype} {tuple(parents.shape)}")
    W = parents.shape[1]
    out_shape = shape if W == K else shape[:batch_dim + 1] + (W,) + shape[batch_dim + 2:]
    if out is None:
        out = torch.zeros(out_shape, dtype=states.dtype, device=states.device)
    elif tuple(out.shape) != out_shape or out.dtype != states.dtype:
        raise _lib.CsError(f"out must be {states.dtype} {out_shape}, got {out.dtype} {tuple(out.shape)}")
    dev = _lib.on_device(states, parents, out)
    if out.numel() == 0:
        return out
    if K == 0:
        raise _lib.CsError("no chains")
    size = states.element_size()
    dst = _rows(out_shape, out.stride(), size, batch_dim)
    if dst is None:
        raise _lib.CsError("out: rows must be adjacent in memory and the leading axes of one stride")
    src = dst if out is states else _rows(shape, states.stride(), size, batch_dim)
    if src is None:   # (never in place: out has the same layout)
        states = states.contiguous()
        src = _rows(shape, states.stride(), size, batch_dim)
    parents = parents.contiguous()
    to, parents_at = out.data_ptr(), parents.data_ptr()
    if parents_at < to + dst[3] and to < parents_at + 8 * B * W:   # parents that are a part of what is written
        parents = parents.clone()
        parents_at = parents.data_ptr()
    _lib.call_on(dev, _lib.lib().cs_beam_reorder, states.data_ptr(), to, src[0], B, K, W, src[2], src[1], dst[1], parents_at)
    return out
