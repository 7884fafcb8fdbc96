"""Plain forms of the beam operators and of the quantised history, in numpy float64 on the CPU."""
import math

import numpy as np


def beam_select(scores, logits, width, *, normalise=True, mask=None, finished=None, end_token=None):
    """scores [B,K] or None, logits [B,K,V], mask [B,K,V] or None -> (scores [B,W] float64, parents, tokens)."""
    x = np.asarray(logits, dtype=np.float64)
    B, K, V = x.shape
    out = np.full((B, width), -np.inf)
    parents = np.tile(np.minimum(np.arange(width), K - 1), (B, 1)).astype(np.int64)
    tokens = np.full((B, width), -1, dtype=np.int64)
    for b in range(B):
        found = []
        for k in range(K):
            before = 0.0 if scores is None else float(scores[b, k])
            if finished is not None and finished[b, k]:
                s = np.full(V, -np.inf)
                s[end_token] = before
            else:
                row = x[b, k] if mask is None else np.where(mask[b, k], x[b, k], -np.inf)
                lse = 0.0
                if normalise:
                    if np.isnan(row).any() or (row == np.inf).any() or not (row > -np.inf).any():
                        continue
                    top = row.max()
                    lse = top + math.log(np.exp(row - top).sum())
                with np.errstate(invalid="ignore"):
                    s = before + (row - lse)
            v = np.flatnonzero(s > -np.inf)    # (a NaN is not)
            # (of one beam only the first W by (score, index) can be among the W best)
            v = v[np.lexsort((v, -s[v]))[:width]]
            found += [(-s[i], k * V + i) for i in v]
        for w, (s, at) in enumerate(sorted(found)[:width]):
            out[b, w], parents[b, w], tokens[b, w] = -s, at // V, at % V
    return out, parents, tokens


def reorder(states, parents):
    """states [outer,B,K,...], parents [B,W] within [0,K) -> [outer,B,W,...]."""
    return np.stack([states[:, b, parents[b]] for b in range(states.shape[1])], axis=1)


E4M3 = sorted([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1])
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(a, grid):
    """The value of ``grid`` (ascending, non-negative; the last bit of a pattern is its place's) nearest to a >= 0, ties to
    the even pattern."""
    grid = np.asarray(grid)
    mid = (grid[1:] + grid[:-1]) / 2
    up, down = np.searchsorted(mid, a, side="right"), np.searchsorted(mid, a, side="left")
    return grid[np.where(up % 2 == 0, up, down)]


def quantised(x, fmt, group):
    """What states x [...,D] (float32 values) read back as from a QuantisedHistory in float32, in float64.  Read in a type of a
    smaller range they are cut to its largest value."""
    x = np.asarray(x, dtype=np.float64)
    D = x.shape[-1]
    out = np.empty_like(x)
    for lo in range(0, D, group):
        g = x[..., lo:lo + group]
        fine = np.isfinite(g)
        v = np.where(fine, g, 0.0)
        top = np.abs(v).max(axis=-1, keepdims=True)
        if fmt == "int8":
            scale = np.maximum((top.astype(np.float32) / np.float32(127)), np.float32(2.0 ** -126)).astype(np.float64)
            r = np.clip(np.rint(v / scale), -127, 127) * scale
            r = np.where(fine, r, np.nan)
        else:
            grid = E4M3 if fmt == "mxfp8" else E2M1
            e = np.full(top.shape, -127)
            for i in range(-126, 128):
                e = np.where(top > grid[-1] * 2.0 ** (i - 1), i, e)
            scale = np.ldexp(1.0, e)
            r = np.copysign(_nearest(np.abs(v) / scale, grid) * scale, v)
            r = np.where(fine, r, np.nan) if fmt == "mxfp8" else np.where(fine.all(axis=-1, keepdims=True), r, np.nan)
        # what a code or a scale rounds up beyond the largest float32 is cut to it (NaN stays)
        r = np.clip(r, -float(np.finfo(np.float32).max), float(np.finfo(np.float32).max))
        out[..., lo:lo + group] = r
    return out
