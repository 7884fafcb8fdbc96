"""Device-resident imputation histories: ``ImputationHistoryQueue`` (LAIR's historical proposals,
irwg/sampling/utils.py:5-68) and the restricted-availability queue of AC-MWG.

The latter is the counterpart of ``ImputationHistoryQueue_with_restrictedavailability``
(irwg/sampling/utils.py:83-237).  The reference keeps the ring ``[T,B,K,D]`` and the per-chain
availability counters on the host and draws one index per chain in a Python double loop; here
both live in HBM, the index draw / gather are fused into the AC-MWG step kernels
(``cs_acmwg_step``) and this class only tracks the two host scalars (``tail_idx``, ``full``)
and exposes the queue's methods for the warm-up phases and for tests.
"""
import ctypes as C

import torch

from .. import _lib


class ImputationHistoryQueue(object):
    """Ring ``[T,B,K,D]`` of past imputations in HBM with the reference's stratified sampling
    (irwg/sampling/utils.py:5-68).  The host tracks ``tail_idx`` / ``full`` and computes the H ring
    slots of a draw (they are common to the batch); the gather of the chosen imputations into the
    proposal set runs on the device (``cs_history_concat``).

    ``storage`` (``int8`` | ``mxfp8`` | ``mxfp4``; no counterpart in the reference): the ring holds the imputations in 8 or 4
    bits (``QuantisedHistory``), for real-valued data whose float32 ring would not fit; slots and chains are drawn as for
    the float32 ring, the historical proposals are what the ring reads back, observed values included.  ``concat_history`` uploads
    its indices by copies that wait for the stream: an iteration of enqueueing and fetching takes 67 us instead of 17 at 512 examples
    of 4 chains, 105 instead of 111 at 65536."""

    def __init__(self, max_history_length, batch_shape, dtype=torch.float32, device="cuda", storage=None):
        if dtype not in (torch.float32, torch.bool) or (storage is not None and dtype == torch.bool):
            raise NotImplementedError(f"history dtype {dtype}" + (f" with storage {storage}" if storage else ""))
        self.max_history_length = int(max_history_length)
        self.tail_idx = -1
        self.full = False
        self.batch_shape = tuple(batch_shape)
        B, K, D = self.batch_shape
        # dtype bool (the reference's queue for binary data, which stores X.bool()): a uint8 ring holding x != 0
        self.u8 = dtype == torch.bool
        self.quantised = None
        if storage is not None:
            self.quantised = QuantisedHistory(self.max_history_length, self.batch_shape, storage, device=device)
            self._chain_ids = None
            return
        self.history_queue = torch.empty((self.max_history_length, B, K, D),
                                         dtype=torch.uint8 if self.u8 else torch.float32, device=device)

    @property
    def history_queue(self):
        """The ring [T,B,K,D], with ``storage`` its records; may be replaced by one of the same shape."""
        return self._history_queue if self.quantised is None else self.quantised.data

    @history_queue.setter
    def history_queue(self, ring):
        if self.quantised is None:
            self._history_queue = ring
        else:
            self.quantised.data = ring

    def __len__(self):
        assert self.tail_idx > -1, 'Queue is empty.'
        return self.tail_idx + 1 if not self.full else self.max_history_length

    def _increment_tail(self):
        self.tail_idx = (self.tail_idx + 1) % self.max_history_length
        if self.tail_idx == self.max_history_length - 1:
            self.full = True

    def enqueue_batch(self, X):
        B, K, D = self.batch_shape
        X = X.to(self.history_queue.device, torch.float32).contiguous()
        self._increment_tail()
        if self.quantised is not None:
            self.quantised.write(X, self.tail_idx)
            return
        fn = _lib.lib().cs_history_enqueue_u8 if self.u8 else _lib.lib().cs_history_enqueue
        _lib.check(fn(_lib.ptr(self.history_queue), None, self.max_history_length, self.tail_idx, 0, _lib.ptr(X), B, K, D,
                      _lib.current_stream()))

    def window_size(self, num_historical_proposals):
        """Exclusive bound of the per-window integer draws (utils.py:33-36)."""
        return len(self) // num_historical_proposals

    def slots_from_window_draws(self, r, num_historical_proposals):
        """Ring slots of the window draws r[H] (utils.py:37-39)."""
        H, w = num_historical_proposals, self.window_size(num_historical_proposals)
        return [int((int(r[h]) + h * w + self.tail_idx) % len(self)) for h in range(H)]

    def concat_history(self, X, slots, *, chain_of_proposal=None, chain_of_example=None, rng=None, out=None):
        """``concat([X, hist_proposals], dim=1)`` of vae_imputation.py:539-545 -> [B,K+H,D]: historical
        proposal h of example b is ring[slots[h], b, chain] with chain = chain_of_proposal[h]
        (sample_history_with_chain_idx_for_each_sample) or one chain per example
        (sample_history: ``chain_of_example`` [B] int64 on the device, or the counter RNG)."""
        B, K, D = self.batch_shape
        H = len(slots)
        Xc = out if out is not None else torch.empty(B, K + H, D, device=X.device, dtype=torch.float32)
        if self.quantised is not None:
            Xc[:, :K] = X
            at = torch.tensor(slots, dtype=torch.int64, device=X.device).expand(B, H)
            if chain_of_proposal is not None:
                chains = torch.tensor([int(c) for c in chain_of_proposal], dtype=torch.int64, device=X.device).expand(B, H)
            elif chain_of_example is not None:
                chains = chain_of_example.to(X.device, torch.int64)[:, None].expand(B, H)
            else:
                chains = self._drawn_chains(H, rng)
            self.quantised.read(at, chains, out=Xc[:, K:])
            return Xc
        i32 = C.c_int32 * H
        cop = i32(*[int(c) for c in chain_of_proposal]) if chain_of_proposal is not None else None
        coe = chain_of_example.to(X.device, torch.int64).contiguous() if chain_of_example is not None else None
        rng = rng if rng is not None else _lib.make_rng(0)
        fn = _lib.lib().cs_history_concat_u8 if self.u8 else _lib.lib().cs_history_concat
        _lib.check(fn(_lib.ptr(X), _lib.ptr(self.history_queue), B, K, D, H, i32(*slots), cop, _lib.ptr(coe), C.byref(rng),
                      _lib.ptr(Xc), _lib.current_stream()))
        return Xc


    def _drawn_chains(self, H, rng):
        """[B,H]: the chain per example that the counter RNG gives ``cs_history_concat``, by that call on a ring of chain
        numbers."""
        B, K, _ = self.batch_shape
        if self._chain_ids is None:
            self._chain_ids = torch.arange(K, device=self.history_queue.device, dtype=torch.float32).expand(1, B, K).contiguous()
        ids, got = self._chain_ids, torch.empty(B, K + 1, device=self.history_queue.device)
        rng = rng if rng is not None else _lib.make_rng(0)
        _lib.check(_lib.lib().cs_history_concat(_lib.ptr(ids), _lib.ptr(ids), B, K, 1, 1, (C.c_int32 * 1)(0), None, None, C.byref(rng),
                                                _lib.ptr(got), _lib.current_stream()))
        return got[:, K:].long().expand(B, H)


def glr_history_chain_idx(K, num_historical_proposals, glr_cluster_size):
    """Chain that every historical proposal is taken from when global-local resampling is combined
    with the history, so that each group only receives history of its own chains
    (vae_imputation.py:505-537)."""
    import math
    H, c = num_historical_proposals, glr_cluster_size
    assert (K + H) % c == 0
    G = (K + H) // c
    assert G <= K
    num_rem = math.ceil(K / G) * G - K
    base = list(range(K)) + list(range(G - num_rem, G))
    chain = base * ((K + H) // len(base))
    if (K + H) % len(base) != 0:
        chain = chain + base[:(K + H) - len(chain)]
    return chain[K:]


class ImputationHistoryQueue_with_restrictedavailability(object):
    def __init__(self, max_history_length, batch_shape, dtype=torch.float32, device="cuda", compact=True):
        if dtype not in (torch.float32, torch.bool):
            raise NotImplementedError(f"history dtype {dtype}")
        self.max_history_length = int(max_history_length)
        self.tail_idx = -1
        self.full = False
        self.bool_data = dtype == torch.bool  # values are 0/1
        # dtype bool (the reference stores X.bool(), test_step_vae_sampling.py:1537-1541): a uint8 ring holding x != 0,
        # a quarter of the float ring (Omniglot, B=200, K=5, T=5000: 3.9 GB instead of 15.7).  compact=False keeps
        # the float ring: the fused MLP encoder reads its input rows as float32 straight from the ring.
        self.u8 = self.bool_data and compact
        self.batch_shape = tuple(batch_shape)
        B, K, D = self.batch_shape
        # t b k d
        self.history_queue = torch.empty((self.max_history_length, B, K, D),
                                         dtype=torch.uint8 if self.u8 else torch.float32, device=device)
        # b k
        self.available_timesteps = torch.zeros((B, K), dtype=torch.int64, device=device)

    def __len__(self):
        assert self.tail_idx > -1, 'Queue is empty.'
        return self.tail_idx + 1 if not self.full else self.max_history_length

    def update_available_timesteps(self, make_full_history_available):
        """BxK boolean tensor (or None = all chains): those chains may use the whole history."""
        mask = make_full_history_available
        m8 = None
        if mask is not None:
            m8 = mask.to(self.available_timesteps.device, torch.uint8).contiguous()
        B, K, _ = self.batch_shape
        _lib.check(_lib.lib().cs_history_set_available(_lib.ptr(self.available_timesteps), _lib.ptr(m8), B * K,
                                                       len(self), _lib.current_stream()))

    def advance(self):
        """Host bookkeeping of one enqueue (utils.py:109-113); returns (new_tail, was_full)."""
        was_full = self.full
        self.tail_idx = (self.tail_idx + 1) % self.max_history_length
        if self.tail_idx == self.max_history_length - 1:
            self.full = True
        return self.tail_idx, was_full

    def enqueue_batch(self, X):
        B, K, D = self.batch_shape
        X = X.to(self.history_queue.device, torch.float32).contiguous()
        new_tail, was_full = self.advance()
        fn = _lib.lib().cs_history_enqueue_u8 if self.u8 else _lib.lib().cs_history_enqueue
        _lib.check(fn(_lib.ptr(self.history_queue), _lib.ptr(self.available_timesteps), self.max_history_length, new_tail,
                      int(was_full), _lib.ptr(X), B, K, D, _lib.current_stream()))

    def slots_from_draws(self, r):
        """Ring slot of integer draws r[B,K] in [0, max(avail,1)) (utils.py:225-232)."""
        if self.full:
            return (r + self.tail_idx + 1) % self.max_history_length
        return r


_STRIDES = C.c_int64 * 3


class QuantisedHistory:
    """Ring ``[T,B,K,D]`` of past states in 8 or 4 bits: quantised as they are written, read back by slot and chain.

    ``fmt``: ``int8`` (a float32 scale for every ``group`` = 32, 64 or 128 consecutive values), ``mxfp8`` / ``mxfp4`` (e4m3 /
    e2m1 elements of OCP Microscaling, groups of 32 with a power of two).  A state is one record, codes and scales
    together (include/csvae.h, cs_qcache): a MiniBooNE state of 43 values takes 48, 48 or 32 bytes instead of 172.  A value
    that is not finite reads as NaN (mxfp4: its whole group).  ``data`` is the ring [T,B,K,record] uint8, zeros at first (they
    read as zeros, in int8; as zeros of the smallest scale in the others)."""

    def __init__(self, max_history_length, batch_shape, fmt, group=None, device="cuda"):
        if fmt not in _lib.CS_QFMT:
            raise NotImplementedError(f"history format {fmt!r}")
        group = (64 if fmt == "int8" else 32) if group is None else int(group)
        self.max_history_length, self.batch_shape, self.fmt, self.group = int(max_history_length), tuple(batch_shape), fmt, group
        B, K, D = self.batch_shape
        if max(self.max_history_length, B, K, D, abs(group)) > _lib.INT32_MAX:
            raise _lib.CsError(f"no history of {self.max_history_length} states {self.batch_shape}: at most 2^31 - 1 of each")
        self.record_bytes = int(_lib.lib().cs_qcache_record_bytes(_lib.CS_QFMT[fmt], group, D))
        if self.record_bytes < 0 or self.max_history_length < 1 or K < 1:
            raise _lib.CsError(f"no history of {self.max_history_length} states {self.batch_shape} as {fmt}, groups of {group}")
        self._describe()
        self.data = torch.zeros((self.max_history_length, B, K, self.record_bytes), dtype=torch.uint8, device=device)

    def _describe(self):
        self._desc = _lib.cs_qcache(None, self.max_history_length, *self.batch_shape, _lib.CS_QFMT[self.fmt], self.group)
        self._ring = C.byref(self._desc)

    # (a copy, shallow or deep, has a descriptor of its own: it names the memory of that copy's ``data``)
    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_desc", "_ring")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._describe()
        self.data = self._data

    @property
    def data(self):
        return self._data

    @data.setter
    def data(self, t):
        if tuple(t.shape) != (self.max_history_length,) + self.batch_shape[:2] + (self.record_bytes,) or t.dtype != torch.uint8 \
                or not t.is_contiguous() or t.data_ptr() % 16:
            raise _lib.CsError("data must be a contiguous uint8 [T,B,K,record], aligned to 16 bytes")
        self._data, self._desc.data = t, t.data_ptr()

    def _int64(self, t, shape, what):
        if t.dtype != torch.int64 or t.shape != shape:
            raise _lib.CsError(f"{what} must be int64 {list(shape)}, got {t.dtype} {list(t.shape)}")
        return t.contiguous()

    def _slot(self, start):
        start = int(start)
        return start % self.max_history_length if start >= 0 else -1   # (which the library refuses)

    def write(self, X, start, counts=None):
        """Quantise ``X`` [n,B,K,D] or [B,K,D] (float32 / bfloat16 / float16, any strides with D adjacent; n <= T) into the
        slots ``start .. start + n - 1`` (mod T).  ``start``: an int, or an int64 tensor [B,K] with a position per chain (negative:
        the chain is left out).  ``counts`` (int64 [B,K]): only the first ``counts[b,k]`` states of a chain are written; all
        other records stay as they are."""
        B, K, D = self.batch_shape
        shape = X.shape
        if shape[-3:] != self.batch_shape or len(shape) not in (3, 4):
            raise _lib.CsError(f"states must be [n,{B},{K},{D}], got {list(shape)}")
        kind = _lib.CS_TYPE.get(X.dtype, 3)
        if kind == 3:
            raise _lib.CsError(f"states must be float32, bfloat16 or float16, got {X.dtype}")
        start_at, first, counts_at = None, 0, None
        if torch.is_tensor(start):
            start = self._int64(start, (B, K), "start")
            start_at = start.data_ptr()
        else:
            first = self._slot(start)
        if counts is not None:
            counts = self._int64(counts, (B, K), "counts")
            counts_at = counts.data_ptr()
        dev = _lib.on_device(self._data, X, start if start_at else None, counts)
        strides = X.stride()
        if strides[-1] != 1 and D > 1:
            X = X.contiguous()
            strides = X.stride()
        _lib.call_on(dev, _lib.lib().cs_qcache_write, self._ring, X.data_ptr(), kind, shape[0] if len(shape) == 4 else 1,
                     _STRIDES(*(strides[:3] if len(shape) == 4 else (0, strides[0], strides[1]))), start_at, first, counts_at)

    def read(self, slots, chains=None, *, dtype=torch.float32, out=None):
        """``out[n,b,j] = state at slots[n,b,j] of chain chains[n,b,j]`` (None: of chain j) of example b, zeros where slot or
        chain do not exist.  ``slots`` / ``chains`` int64 [N,B,J] or [B,J]; ``out`` [N,B,J,D] (or [B,J,D]): any strides with D
        adjacent.  A value beyond the range of the type that is read becomes the type's largest (a finite state never reads as an
        infinity)."""
        B, K, D = self.batch_shape
        shape = tuple(slots.shape)
        if len(shape) not in (2, 3) or shape[-2] != B or slots.dtype != torch.int64 or (chains is None and shape[-1] != K) \
                or shape[-1] > _lib.INT32_MAX:
            raise _lib.CsError(f"slots must be int64 [N,{B},{K}] (or [N,{B},J] with chains), got {slots.dtype} {list(shape)}")
        chains_at = None
        if chains is not None:
            chains = self._int64(chains, shape, "chains")
            chains_at = chains.data_ptr()
        slots = slots.contiguous()
        out, kind, strides = self._out(out, shape + (D,), dtype)
        if out.numel():
            dev = _lib.on_device(self._data, slots, chains, out)
            single = len(shape) == 2
            _lib.call_on(dev, _lib.lib().cs_qcache_read, self._ring, slots.data_ptr(), 0, chains_at, 1 if single else shape[0],
                         shape[-1], out.data_ptr(), kind, _STRIDES(*((0,) + strides[:2] if single else strides[:3])))
        return out

    def read_steps(self, start, n, *, dtype=torch.float32, out=None):
        """The states of all chains at the slots ``start .. start + n - 1`` (mod T): [n,B,K,D]."""
        B, K, D = self.batch_shape
        out, kind, strides = self._out(out, (int(n), B, K, D), dtype)
        if out.numel():
            dev = _lib.on_device(self._data, out)
            _lib.call_on(dev, _lib.lib().cs_qcache_read, self._ring, None, self._slot(start), None, int(n), K, out.data_ptr(), kind,
                         _STRIDES(*strides[:3]))
        return out

    def _out(self, out, shape, dtype):
        """(the tensor to read into, its element type, its strides)"""
        if out is None:
            kind = _lib.CS_TYPE.get(dtype, 3)
            if kind == 3:
                raise _lib.CsError(f"states are read as float32, bfloat16 or float16, got {dtype}")
            out = torch.empty(shape, dtype=dtype, device=self._data.device)
            return out, kind, out.stride()
        kind, strides = _lib.CS_TYPE.get(out.dtype, 3), out.stride()
        if out.shape != shape or kind == 3 or (strides[-1] != 1 and shape[-1] > 1) \
                or any(s == 0 and n > 1 for s, n in zip(strides, shape)):
            raise _lib.CsError(f"out must be float32, bfloat16 or float16 {list(shape)} with adjacent values, every row a place "
                               "of its own")
        return out, kind, strides

    def reorder(self, parents, steps=None):
        """The records of every chain follow ``parents`` [B,K] in place (``beam.reorder_states``: K <= 64), in the first ``steps``
        slots (None: all)."""
        from .beam import reorder_states
        if steps is not None and int(steps) < 0:
            raise _lib.CsError(f"negative number of steps {steps}")
        data = self._data if steps is None else self._data[:int(steps)]
        reorder_states(data, parents, batch_dim=1, out=data)
