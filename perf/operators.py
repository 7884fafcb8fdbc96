"""Timed cases of the beam operators and the quantised history.

Chains are beams here: a state is kept per (example b, chain k).  Four operators: the selection of the best continuations
of all beams of an example (``beam_select``), the reordering of what is kept per chain by the chosen parents
(``reorder_states``), and the history ring in 8 or 4 bits, written (``QuantisedHistory.write``) and read back
(``QuantisedHistory.read``).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---- cases -------------------------------------------------------------------------------------------------------
def _select(B, K, V, W, dtype, masked=False, finished=False, **kw):
    return dict(op="select", B=B, K=K, V=V, W=W, dtype=dtype, masked=masked, finished=finished, **kw)


def _reorder(outer, B, K, W, inner, kind, moved, in_place, **kw):
    return dict(op="reorder", outer=outer, B=B, K=K, W=W, inner=inner, kind=kind, moved=moved, in_place=in_place, **kw)


def _cache(fmt, group, dtype, T, B, K, D, n, N, ragged=False, chains=False, **kw):
    return dict(op="cache", fmt=fmt, group=group, dtype=dtype, T=T, B=B, K=K, D=D, n=n, N=N, ragged=ragged, chains=chains, **kw)


def listed():
    return [
        # one example searched by itself, token by token: latency of a call
        _select(1, 4, 16384, 4, "bf16", name="select_one_example"),
        # a served batch: float32 logits, an odd vocabulary, a constraint on the next value, some beams at their end
        _select(24, 6, 50021, 6, "f32", masked=True, finished=True, name="select_constrained"),
        # a large batch over a long vocabulary
        _select(64, 16, 131072, 16, "bf16", name="select_long_vocabulary"),
        # the best 5 of the 600 x 17 proposals that a HEPMASS run with 16 chains keeps per example (no beams before it)
        _select(4096, 1, 10200, 5, "f32", name="select_final_proposals"),
        # latents of a MiniBooNE batch follow their ancestors: latency of a call
        _reorder(1, 512, 4, 4, 32, "f32", 4, False, name="reorder_latents"),
        # a MiniBooNE history of 600 iterations, in place, half of the chains replaced by copies of survivors
        _reorder(600, 512, 4, 4, 43, "f32", 2, True, name="reorder_history"),
        # a binary history of 28 x 28 images, in place
        _reorder(500, 200, 5, 5, 784, "u8", 2, True, name="reorder_binary_history"),
        # one iteration of a MiniBooNE chain: keep this state, fetch one past state per chain
        _cache("int8", 64, "f32", 1000, 256, 5, 43, 1, 1, name="cache_one_step"),
        # fetching past states of every chain of a HEPMASS batch, from any of its chains, for a set of proposals
        _cache("int8", 32, "f32", 600, 512, 16, 21, 1, 64, chains=True, name="cache_fetch_proposals"),
        # a long stretch kept at once and read back, 8-bit floats
        _cache("mxfp8", 32, "bf16", 2048, 8, 8, 128, 2048, 2048, name="cache_stretch"),
        # sequences of different lengths at different positions, 4 bits, an odd width
        _cache("mxfp4", 32, "f16", 512, 16, 4, 1001, 300, 300, ragged=True, name="cache_ragged"),
        # the largest: wide states of a large batch
        _cache("mxfp8", 32, "bf16", 1024, 32, 4, 1024, 1024, 1024, name="cache_wide"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "cache", "cache"])
    if op == "select":
        B, K, V = _log(rng, 1, 64), rng.randint(1, 16), _log(rng, 500, 131072)
        return _select(B, K, V, rng.randint(1, 16), rng.choice(list(DTYPES)), rng.random() < 0.4, rng.random() < 0.4)
    if op == "reorder":
        outer, B, K, inner = _log(rng, 1, 400), _log(rng, 1, 512), rng.randint(2, 16), _log(rng, 8, 1024)
        kind = rng.choice(["f32", "bf16", "u8"])
        while outer * B * K * inner > 1 << 27:
            outer = max(1, outer // 2)
            B = max(1, B // 2)
        if rng.random() < 0.5:
            return _reorder(outer, B, K, K, inner, kind, rng.randint(1, K // 2), True)
        W = rng.randint(1, 16)
        return _reorder(outer, B, K, W, inner, kind, W, False)
    fmt = rng.choice(["int8", "mxfp8", "mxfp4"])
    group = rng.choice([32, 64, 128]) if fmt == "int8" else 32
    T, B, K, D = _log(rng, 16, 1024), _log(rng, 1, 256), rng.randint(1, 16), _log(rng, 8, 1024)
    while T * B * K * D > 1 << 26:
        T = max(2, T // 2)
        B = max(1, B // 2)
    ragged = rng.random() < 0.4
    n = max(1, min(T, _log(rng, 1, T)))
    N = n if ragged else max(1, min(T, _log(rng, 1, T)))
    return _cache(fmt, group, rng.choice(list(DTYPES)), T, B, K, D, n, N, ragged, not ragged and rng.random() < 0.4)


def _record_bytes(c):
    groups = -(-c["D"] // c["group"])
    return {"int8": 4 * groups + c["D"], "mxfp8": groups + c["D"], "mxfp4": groups + (c["D"] + 1) // 2}[c["fmt"]]


def work(c):
    if c["op"] == "select":
        n = c["B"] * c["K"] * c["V"]
        # an exponential of 64 bits per value is priced at 12 operations
        return {"bytes": n * BYTES[c["dtype"]] + (c["B"] * c["V"] if c["masked"] else 0) + 20 * c["B"] * c["W"] + 5 * c["B"] * c["K"],
                "flops": 12 * n}
    if c["op"] == "reorder":
        row = c["inner"] * {"f32": 4, "bf16": 2, "u8": 1}[c["kind"]]
        if c["in_place"]:   # the moved rows and as many distinct sources
            moved, read = c["moved"], c["moved"]
        else:               # random ancestors: the expected number of distinct ones
            moved, read = c["W"], c["K"] * (1 - (1 - 1 / c["K"]) ** c["W"])
        return {"bytes": c["outer"] * c["B"] * row * (moved + read) + 8 * c["B"] * c["W"], "flops": 0}
    chains = c["B"] * c["K"]
    wrote, took = c["n"] * chains, c["N"] * chains
    if c["ragged"]:         # counts are uniform in [0, n]
        wrote, took = wrote / 2, took / 2
    row = c["D"] * BYTES[c["dtype"]]
    return {"bytes": wrote * (row + _record_bytes(c)) + took * _record_bytes(c) + c["N"] * chains * row
            + 8 * c["N"] * chains * (2 if c["chains"] else 1), "flops": 4 * (wrote + took) * c["D"]}


# ---- inputs ------------------------------------------------------------------------------------------------------
class State:
    pass


def _states(shape, gen, dtype):
    """Standardised features: every column with a scale and an offset of its own, now and then a far value."""
    D = shape[-1]
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(0.8 * torch.randn(D, generator=gen, device="cuda"))
    x += 0.3 * torch.randn(D, generator=gen, device="cuda")
    return x.to(dtype)


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    ints = lambda lo, hi, shape: torch.randint(lo, hi, shape, generator=gen, device="cuda")  # noqa: E731
    s = State()
    s.c = c
    if c["op"] == "select":
        B, K, V = c["B"], c["K"], c["V"]
        s.logits = torch.empty(B, K, V, device="cuda", dtype=DTYPES[c["dtype"]])
        for b in range(0, B, max(1, (1 << 24) // (K * V))):   # (made in pieces: the float32 normals are larger than the logits)
            part = s.logits[b:b + max(1, (1 << 24) // (K * V))]
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * 2.5)
        s.scores = None if K == 1 and not c["finished"] else torch.sort(-6 - 2 * torch.rand(B, K, generator=gen, device="cuda"), dim=1, descending=True).values
        s.mask = torch.rand(B, 1, V, generator=gen, device="cuda") < 0.7 if c["masked"] else None
        s.finished = torch.rand(B, K, generator=gen, device="cuda") < 0.2 if c["finished"] else None
        s.end_token = 2 if c["finished"] else None
        return s
    if c["op"] == "reorder":
        outer, B, K, W = c["outer"], c["B"], c["K"], c["W"]
        shape = (outer, B, K, c["inner"])
        if c["kind"] == "u8":
            s.states = ints(0, 2, shape).to(torch.uint8)
        else:
            s.states = _states(shape, gen, DTYPES[c["kind"]])
        if c["in_place"]:
            # survivors keep their slot and the others become copies of different survivors, as a search arranges it
            order = torch.rand(B, K, generator=gen, device="cuda").argsort(dim=1)
            m = c["moved"]
            s.parents = torch.arange(K, device="cuda").repeat(B, 1)
            s.parents.scatter_(1, order[:, :m], order[:, m:2 * m])
            s.out = None
        else:
            s.parents = ints(0, K, (B, W))
            s.out = torch.zeros(outer, B, W, c["inner"], device="cuda", dtype=s.states.dtype)
        return s
    T, B, K, D, n, N = c["T"], c["B"], c["K"], c["D"], c["n"], c["N"]
    dt = DTYPES[c["dtype"]]
    if own:
        from vae_conditional_sampling_amd.sampling.utils import QuantisedHistory
        s.cache = QuantisedHistory(T, (B, K, D), c["fmt"], group=c["group"], device="cuda")
    else:
        s.cache = PlainHistory(T, B, K, D, c["fmt"], c["group"])
    if n < T:   # a program reads what it kept before
        old = _states((T, B, K, D), gen, dt)
        s.cache.write(old, 0)
        s.old = old if c.get("with_old") else None
        del old
    s.x = _states((n, B, K, D), gen, dt)
    if c["ragged"]:
        s.start = ints(0, T, (B, K))
        s.counts = ints(0, n + 1, (B, K))
        i = torch.arange(n, device="cuda")[:, None, None]
        s.slots = torch.where(i < s.counts, (s.start + i) % T, -1)
        s.chains = None
    else:
        s.start, s.counts = int(ints(0, T, (1,))), None
        if N == n == T:
            s.slots = ((s.start + torch.arange(n, device="cuda")) % T)[:, None, None].expand(n, B, K).contiguous()
        else:
            s.slots = ints(0, T, (N, B, K))
        s.chains = ints(0, K, (N, B, K)) if c["chains"] else None
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------
def _select_plain(s):
    B, K, V, W = (s.c[k] for k in "BKVW")
    x = s.logits.double()
    if s.mask is not None:
        x = torch.where(s.mask, x, -math.inf)
    top = x.amax(dim=2, keepdim=True)
    lse = (top + (x - torch.where(top.isinf(), 0.0, top)).exp().sum(dim=2, keepdim=True).log())
    before = torch.zeros(B, K, 1, device="cuda", dtype=torch.float64) if s.scores is None else s.scores.double()[:, :, None]
    v = x + (before - lse)
    if s.finished is not None:
        end = torch.arange(V, device="cuda") == s.end_token
        v = torch.where(s.finished[:, :, None], torch.where(end, before, -math.inf), v)
    v = torch.where(v.isnan(), -math.inf, v).reshape(B, K * V)
    del x
    # the W largest, of equal ones those with the lowest index: everything above the W-th largest value, and the first of those equal to it
    edge = v.topk(W, dim=1).values[:, -1:]
    equal = v == edge
    chosen = (v > edge) | (equal & (equal.cumsum(dim=1) <= W - (v > edge).sum(dim=1, keepdim=True)))
    place = K * V - torch.arange(K * V, device="cuda")
    index = K * V - (chosen * place).topk(W, dim=1).values            # ascending
    value, order = v.gather(1, index).sort(dim=1, descending=True, stable=True)
    index = index.gather(1, order)
    none = value == -math.inf
    slot = torch.arange(W, device="cuda").clamp(max=K - 1)
    return {"scores": value.float(), "parents": torch.where(none, slot, index // V), "tokens": torch.where(none, -1, index % V)}


def _power(e):
    """2^e exactly, from the bits (pow and ldexp of this device's library are an ulp off for some exponents)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


class PlainHistory:
    """The quantised ring by elementary operations: codes and scales in tensors of their own."""

    def __init__(self, T, B, K, D, fmt, group):
        self.T, self.B, self.K, self.D, self.fmt, self.group = T, B, K, D, fmt, group
        self.groups = -(-D // group)
        self.codes = torch.zeros(T, B, K, D, device="cuda", dtype=torch.int8)
        self.scales = torch.zeros(T, B, K, self.groups, device="cuda")

    def encode(self, x):
        """codes [..., D] as int8 (of e4m3: its bits; of e2m1: twice the value) and scales [..., groups]."""
        x = torch.nn.functional.pad(x.double(), (0, self.groups * self.group - self.D))
        x = x.reshape(*x.shape[:-1], self.groups, self.group)
        fine = x.isfinite()
        top = torch.where(fine, x, 0.0).abs().amax(dim=-1, keepdim=True)
        if self.fmt == "int8":
            scale = (top / 127).float().clamp(min=2.0 ** -126)
            codes = torch.where(fine, (x / scale.double()).round().clamp(-127, 127), -128.0).to(torch.int8)
        else:
            largest, low, bits = (448.0, -6, 3) if self.fmt == "mxfp8" else (6.0, 0, 1)
            f, e = torch.frexp(top)
            limit = math.frexp(largest)
            e = torch.where(top > 0, e - limit[1] + (f > limit[0]), -127).clamp(-127, 127)
            y = x * _power(-e)
            step = _power((torch.frexp(y)[1] - 1).clamp(min=low) - bits)
            y = torch.where(fine, (y / step).round() * step, math.nan)
            scale = _power(e).float()
            if self.fmt == "mxfp8":
                codes = y.float().to(torch.float8_e4m3fn).view(torch.int8)
            else:
                scale = torch.where(fine.all(dim=-1, keepdim=True), scale, math.nan)
                codes = torch.where(fine, 2 * y, 0.0).to(torch.int8)
        return codes.reshape(*codes.shape[:-2], -1)[..., :self.D], scale[..., 0]

    def write(self, x, start, counts=None):
        i = torch.arange(x.shape[0], device="cuda")[:, None, None]
        b = torch.arange(self.B, device="cuda")[:, None]
        k = torch.arange(self.K, device="cuda")
        at = (start + i) % self.T
        at = at.expand(x.shape[0], self.B, self.K)
        codes, scales = self.encode(x)
        if counts is not None:
            kept = (i < counts)[..., None]
            codes = torch.where(kept, codes, self.codes[at, b, k])
            scales = torch.where(kept, scales, self.scales[at, b, k])
        self.codes[at, b, k] = codes
        self.scales[at, b, k] = scales

    def read(self, slots, chains=None, dtype=torch.float32):
        b = torch.arange(self.B, device="cuda")[:, None]
        k = torch.arange(self.K, device="cuda") if chains is None else chains
        there = (slots >= 0) & (slots < self.T)
        at = torch.where(there, slots, 0)
        codes = self.codes[at, b, k]
        scale = self.scales[at, b, k].repeat_interleave(self.group, dim=-1)[..., :self.D]
        if self.fmt == "int8":
            value = torch.where(codes == -128, math.nan, codes.float())
        elif self.fmt == "mxfp8":
            value = codes.view(torch.float8_e4m3fn).float()
        else:
            value = codes.float() / 2
        big = torch.finfo(torch.float32).max
        return torch.where(there[..., None], (value * scale).clamp(-big, big), 0.0).to(dtype)


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(s):
    c = s.c
    if c["op"] == "select":
        if own:
            from vae_conditional_sampling_amd.sampling.beam import beam_select
            step = beam_select(s.scores, s.logits, c["W"], mask=s.mask, finished=s.finished, end_token=s.end_token)
            return {"scores": step.scores, "parents": step.parents, "tokens": step.tokens}
        return _select_plain(s)
    if c["op"] == "reorder":
        if own:
            from vae_conditional_sampling_amd.sampling.beam import reorder_states
            return reorder_states(s.states, s.parents, batch_dim=1, out=s.states if c["in_place"] else s.out)
        b = torch.arange(c["B"], device="cuda")[:, None]
        moved = s.states[:, b, s.parents]
        return (s.states if c["in_place"] else s.out).copy_(moved)
    s.cache.write(s.x, s.start, s.counts)
    return s.cache.read(s.slots, s.chains, dtype=DTYPES[c["dtype"]])


# ---- in 64 bits --------------------------------------------------------------------------------------------------
def _select_exact(s):
    B, K, V, W = (s.c[k] for k in "BKVW")
    scores, index = [], []
    for b in range(B):
        x = s.logits[b].double()
        if s.mask is not None:
            x = x.masked_fill(~s.mask[b], -math.inf)
        p = x - torch.logsumexp(x, dim=1, keepdim=True)
        if s.scores is not None:
            p = p + s.scores[b].double()[:, None]
        if s.finished is not None:
            for k in s.finished[b].nonzero()[:, 0].tolist():
                p[k] = -math.inf
                p[k, s.end_token] = float(s.scores[b, k])
        value, at = torch.sort(p.reshape(-1), descending=True, stable=True)
        scores.append(value[:W])
        index.append(at[:W])
    scores, index = torch.stack(scores), torch.stack(index)
    return {"scores": scores, "parents": index // V, "tokens": index % V}


def _grid(fmt):
    """The non-negative values that an element can hold, ascending."""
    if fmt == "mxfp4":
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    values = [m / 8 * 2.0 ** -6 for m in range(8)]
    values += [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return values[:-1]   # (the last pattern is NaN)


def _cache_values(x, fmt, group):
    """What the rows x [..., D] read back as, in 64 bits."""
    parts = []
    for lo in range(0, x.shape[-1], group):
        g = x[..., lo:lo + group].double()
        top = g.abs().amax(dim=-1, keepdim=True)
        if fmt == "int8":
            scale = torch.from_numpy(np.maximum((top.cpu().numpy() / 127).astype(np.float32), np.float32(2.0 ** -126))).cuda().double()
            q = g / scale
            low = q.floor()
            up = (q - low > 0.5) | ((q - low == 0.5) & (low % 2 != 0))
            parts.append((low + up).clamp(-127, 127) * scale)
        else:
            grid = torch.tensor(_grid(fmt), device="cuda", dtype=torch.float64)
            powers = torch.tensor([math.ldexp(1.0, e) for e in range(-127, 128)], device="cuda", dtype=torch.float64)
            scale = powers[torch.bucketize(top, grid[-1] * powers).clamp(max=254)]   # the smallest power with top in its range
            a = g.abs() / scale
            between = (grid[1:] + grid[:-1]) / 2
            up, down = torch.bucketize(a, between, right=True), torch.bucketize(a, between)   # they differ on a border
            parts.append(grid[torch.where(up % 2 == 0, up, down)] * g.sign() * scale)
    return torch.cat(parts, dim=-1)


def exact(c, seed):
    s = prepare(dict(c, with_old=True), seed)
    if c["op"] == "select":
        return _select_exact(s)
    if c["op"] == "reorder":
        at = s.parents[None, :, :, None].expand(c["outer"], c["B"], c["W"], c["inner"])
        got = torch.take_along_dim(s.states, at, dim=2)
        return got.double() if c["kind"] != "u8" else got
    if c["ragged"]:
        i = torch.arange(c["n"], device="cuda")[:, None, None, None]
        return torch.where(i < s.counts[..., None], _cache_values(s.x, c["fmt"], c["group"]), 0.0)
    ring = torch.zeros(c["T"], c["B"], c["K"], c["D"], device="cuda", dtype=s.x.dtype)
    if c["n"] < c["T"]:
        ring.copy_(s.old)
    ring[(s.start + torch.arange(c["n"], device="cuda")) % c["T"]] = s.x
    b = torch.arange(c["B"], device="cuda")[:, None]
    k = torch.arange(c["K"], device="cuda") if s.chains is None else s.chains
    return _cache_values(ring[s.slots, b, k], c["fmt"], c["group"])
