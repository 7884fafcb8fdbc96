"""beam_select and reorder_states against plain forms in float64 (oracle/cs_oracle_beam.py).  Indices are exact; a score is
the 64-bit value rounded once, off by at most half a step of its type (2^-24 relative in float32); the kernel's 64-bit
value itself is off by the summation of the normaliser: 1e-10 absolute covers 2^17 terms of relative error below 4e-11."""
import math

import numpy as np
import pytest
import torch

from oracle import cs_oracle_beam as O
from vae_conditional_sampling_amd import _lib
from vae_conditional_sampling_amd.sampling.beam import beam_select, reorder_states

pytestmark = pytest.mark.gpu

SUM = 1e-10


def host(t):
    return t.double().cpu().numpy()


def check(step, scores, logits, width, *, normalise=True, mask=None, finished=None, end_token=None):
    full = None if mask is None else np.broadcast_to(mask.bool().cpu().numpy(), logits.shape)
    ref = O.beam_select(None if scores is None else host(scores), host(logits), width, normalise=normalise, mask=full,
                        finished=None if finished is None else finished.cpu().numpy(), end_token=end_token)
    got = host(step.scores)
    assert step.scores.dtype == (torch.float32 if scores is None else scores.dtype)
    assert np.array_equal(step.parents.cpu().numpy(), ref[1]), "parents"
    assert np.array_equal(step.tokens.cpu().numpy(), ref[2]), "tokens"
    fine = np.isfinite(ref[0])
    assert np.array_equal(got[~fine], ref[0][~fine])
    half = 2.0 ** -24 if step.scores.dtype == torch.float32 else 2.0 ** -53
    assert (np.abs(got[fine] - ref[0][fine]) <= half * np.abs(ref[0][fine]) + SUM * (1 + half)).all()


def make(B, K, V, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(B, K, V, generator=g) * scale).to(dtype).cuda()
    scores = (-5 - 2 * torch.rand(B, K, generator=g)).cuda()
    return scores, logits, g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,K,V,W", [(1, 1, 1, 1), (1, 1, 1, 64), (2, 3, 2, 4), (3, 1, 63, 5), (2, 4, 64, 8), (2, 2, 65, 64), (1, 5, 2047, 16),
                                     (2, 2, 2048, 3), (1, 3, 2049, 32), (2, 17, 500, 17), (1, 2, 50021, 64), (1, 4, 16384, 4),
                                     (5, 1, 10200, 5), (1, 300, 7, 20), (1, 2048, 3, 64)])
def test_selection(dtype, B, K, V, W):
    scores, logits, _ = make(B, K, V, dtype, 100 * K + V)
    check(beam_select(scores, logits, W), scores, logits, W)
    check(beam_select(None, logits, W), None, logits, W)
    s64 = scores.double() - 1e-9
    check(beam_select(s64, logits, W), s64, logits, W)
    check(beam_select(scores, logits, W, normalise=False), scores, logits, W, normalise=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [5, 64, 2049, 6001])
def test_masks_and_finished_beams(dtype, V):
    B, K, W, end = 3, 5, 6, V // 2
    scores, logits, g = make(B, K, V, dtype, V)
    mask = (torch.rand(B, K, V, generator=g) < 0.5).cuda()
    mask[0, 1] = False                      # a beam without a value
    mask[1] = False                         # an example without one
    mask[2, 0, :] = False
    mask[2, 0, V - 1] = True                # one value left
    wild = logits.masked_fill(~mask, float("nan"))   # what is not allowed may hold anything
    wild[:, 2][~mask[:, 2]] = float("inf")
    wild[:, 3][~mask[:, 3]] = torch.finfo(dtype).min
    check(beam_select(scores, wild, W, mask=mask), scores, wild, W, mask=mask)
    shared = mask[2, 1]                     # one mask for all, and one per example
    check(beam_select(scores, logits, W, mask=shared), scores, logits, W, mask=shared)
    check(beam_select(scores, logits, W, mask=mask[:, 2:3]), scores, logits, W, mask=mask[:, 2:3])
    check(beam_select(scores, logits, W, mask=shared.view(torch.uint8)), scores, logits, W, mask=shared)
    finished = torch.zeros(B, K, dtype=torch.bool)
    finished[0, 1] = finished[1, :] = finished[2, 4] = True
    finished = finished.cuda()
    gone = wild.clone()
    gone[finished] = float("nan")
    kw = dict(mask=mask, finished=finished, end_token=end)
    check(beam_select(scores, gone, W, **kw), scores, gone, W, **kw)
    with pytest.raises(_lib.CsError, match="end_token"):
        beam_select(scores, logits, W, finished=finished)
    with pytest.raises(_lib.CsError, match="end token"):
        beam_select(scores, logits, W, finished=finished, end_token=V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_equal_values_go_to_the_lowest_index(dtype):
    for B, K, V, W in ((2, 3, 5000, 16), (1, 64, 64, 16), (1, 1, 4096, 64), (1, 200, 70, 64)):
        logits = torch.zeros(B, K, V, dtype=dtype, device="cuda")      # everything equal: more than any list holds
        scores = torch.zeros(B, K, device="cuda")
        for normalise in (True, False):
            check(beam_select(scores, logits, W, normalise=normalise), scores, logits, W, normalise=normalise)
        logits[:, K // 2, V // 3:] = 1.0                               # a long stretch of equal ones
        check(beam_select(scores, logits, W), scores, logits, W)
        logits[:, :, V // 2] = -0.0                                    # the zeros are one
        check(beam_select(scores, logits, W, normalise=False), scores, logits, W, normalise=False)
    rising = torch.arange(3000, dtype=torch.float32).floor_divide(3).div(256)
    for row in (rising, rising.flip(0)):                               # along a lane's values
        logits = row.to(dtype).repeat(2, 2, 1).cuda()
        check(beam_select(None, logits, 48), None, logits, 48)
    two = torch.randn(1, 1, 3000, generator=torch.Generator().manual_seed(1)).to(dtype).cuda().repeat(1, 2, 1)   # twin beams
    check(beam_select(torch.zeros(1, 2, device="cuda"), two, 7), torch.zeros(1, 2), two, 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_values_that_are_not_finite(dtype):
    inf, nan = float("inf"), float("nan")
    scores, logits, g = make(4, 4, 3000, dtype, 5)
    logits[0, 0, 7] = nan
    logits[0, 1, 2999] = inf
    logits[0, 2] = -inf
    logits[1, 0, ::2] = -inf
    logits[1, 1, :2048] = nan               # a whole stretch
    logits[1, 2, 2048:] = -inf
    logits[2, 3] = torch.finfo(dtype).min
    logits[2, 2] = torch.finfo(dtype).max
    scores[3, 1], scores[3, 2], scores[3, 3] = -inf, nan, -inf
    for W in (1, 9):
        check(beam_select(scores, logits, W), scores, logits, W)
        check(beam_select(scores, logits, W, normalise=False), scores, logits, W, normalise=False)
    dead = torch.full((4, 4), -inf, device="cuda")
    step = beam_select(dead, logits, 6)
    assert (step.scores == -inf).all() and (step.tokens == -1).all()
    assert torch.equal(step.parents.cpu(), torch.tensor([0, 1, 2, 3, 3, 3]).repeat(4, 1))
    far = torch.zeros(1, 1, 5000, dtype=dtype, device="cuda")          # terms that vanish beside the largest
    far[0, 0, 4321] = 1000.0
    check(beam_select(None, far, 2), None, far, 2)


def test_strides_and_empty_batches():
    scores, logits, g = make(3, 4, 600, torch.float32, 9)
    wide = torch.randn(3, 4, 1300, generator=g).cuda()
    for view in (wide[:, :, 1:601], wide[:, ::2, 3:602], wide[1:2].expand(3, 4, 1300), wide.transpose(0, 1)[:3, :3, 5:],
                 wide[:, :, ::2]):
        s = scores[:view.shape[0], :view.shape[1]]
        check(beam_select(s, view, 5), s, view, 5)
        h = view.bfloat16()
        check(beam_select(s, h, 5), s, h, 5)
    odd = torch.randn(2, 3, 999, generator=g).half().cuda()[:, :, 1:]   # rows at odd 2-byte addresses
    check(beam_select(None, odd, 5), None, odd, 5)
    empty = beam_select(scores[:0], logits[:0], 5)
    assert empty.scores.shape == (0, 5) and empty.parents.shape == (0, 5)


def test_two_selections_at_once_and_repeatability():
    scores, logits, _ = make(4, 6, 40000, torch.bfloat16, 3)
    s2, l2, _ = make(2, 3, 9001, torch.float32, 4)
    alone = beam_select(scores, logits, 6), beam_select(s2, l2, 9)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, (st, a) in enumerate(zip(streams, ((scores, logits, 6), (s2, l2, 9)))):
            with torch.cuda.stream(st):
                got[i].append(beam_select(*a))
    torch.cuda.synchronize()
    for one, many in zip(alone, got):
        for step in many:
            assert all(torch.equal(a, b) for a, b in zip(one, step))


KINDS = [torch.float32, torch.bfloat16, torch.uint8, torch.int64, torch.bool]


def fill(shape, dtype, g):
    x = torch.randint(0, 256, shape, generator=g)
    return (x % 2).bool() if dtype == torch.bool else x.to(dtype)


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("outer,B,K,W,inner", [(1, 1, 1, 1, 1), (1, 5, 4, 4, 32), (7, 3, 4, 4, 43), (3, 2, 5, 5, 784), (2, 3, 16, 16, 12),
                                               (1, 2, 33, 33, 8), (2, 2, 64, 64, 5), (300, 1, 2, 2, 3), (2, 3, 6, 9, 17), (3, 2, 70, 4, 16),
                                               (1, 2, 3, 100, 1), (70000, 1, 2, 2, 1)])
def test_reordering(dtype, outer, B, K, W, inner):
    g = torch.Generator().manual_seed(outer + inner)
    x = fill((outer, B, K, inner), dtype, g)
    parents = torch.randint(0, K, (B, W), generator=g)
    ref = torch.from_numpy(O.reorder(x.numpy() if dtype != torch.bfloat16 else x.float().numpy(), parents.numpy())).to(dtype)
    assert torch.equal(reorder_states(x.cuda(), parents.cuda(), batch_dim=1).cpu(), ref)
    if W == K:
        every = [parents, torch.arange(K).repeat(B, 1), torch.arange(K).flip(0).repeat(B, 1), (torch.arange(K) + 1).remainder(K).repeat(B, 1)]
        for p in every if K <= 64 else ():
            y = x.cuda()
            assert reorder_states(y, p.cuda(), batch_dim=1, out=y) is y
            ref = torch.from_numpy(O.reorder(x.numpy() if dtype != torch.bfloat16 else x.float().numpy(), p.numpy())).to(dtype)
            assert torch.equal(y.cpu(), ref)


def test_rows_without_a_parent_stay():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(6, 4, 5, 9, generator=g).cuda()
    p = torch.tensor([[0, -1, 1, 5, 2], [4, 4, 4, 4, 4], [-1, -1, -1, -1, -1], [1, 0, 3, 2, 1 << 40]]).cuda()
    kept = torch.randn(6, 4, 5, 9, generator=g).cuda()
    out = kept.clone()
    reorder_states(x, p, batch_dim=1, out=out)
    y = x.clone()
    reorder_states(y, p, batch_dim=1, out=y)
    new = reorder_states(x, p, batch_dim=1)
    for b in range(4):
        for w in range(5):
            parent = int(p[b, w])
            there = 0 <= parent < 5
            assert torch.equal(out[:, b, w], x[:, b, parent] if there else kept[:, b, w])
            assert torch.equal(y[:, b, w], x[:, b, parent] if there else x[:, b, w])
            assert torch.equal(new[:, b, w], x[:, b, parent] if there else torch.zeros(6, 9, device="cuda"))


def test_views_and_refusals():
    g = torch.Generator().manual_seed(3)
    big = torch.randn(5, 6, 7, 40, generator=g).cuda()
    p = torch.randint(0, 7, (6, 7), generator=g).cuda()
    ref = torch.from_numpy(O.reorder(big.cpu().numpy(), p.cpu().numpy())).cuda()
    part = big.clone()
    reorder_states(part[1:4, :, :, 3:20], p, batch_dim=1, out=part[1:4, :, :, 3:20])     # a window, in place
    assert torch.equal(part[1:4, :, :, 3:20], ref[1:4, :, :, 3:20])
    part[1:4, :, :, 3:20] = big[1:4, :, :, 3:20]
    assert torch.equal(part, big)                                                        # and nothing around it
    apart = big.transpose(0, 1).contiguous().transpose(0, 1)                             # examples outermost in memory
    assert torch.equal(reorder_states(apart, p, batch_dim=1), ref)
    rows = big.transpose(2, 3).contiguous().transpose(2, 3)                              # a row is not adjacent: copied first
    assert torch.equal(reorder_states(rows, p, batch_dim=1), ref)
    two = big.reshape(5, 6, 7, 8, 5)
    assert torch.equal(reorder_states(two, p, batch_dim=1), ref.reshape(5, 6, 7, 8, 5))
    lead = big.reshape(5, 1, 6, 7, 40).expand(5, 2, 6, 7, 40)                            # shared states, two leading axes
    assert torch.equal(reorder_states(lead, p, batch_dim=2), ref[:, None].expand(5, 2, 6, 7, 40))
    flat = torch.randn(6, 7, generator=g).cuda()
    assert torch.equal(reorder_states(flat, p), flat.gather(1, p))
    assert reorder_states(big[:, :0], p[:0], batch_dim=1).shape == (5, 0, 7, 40)
    assert reorder_states(big[:0], p, batch_dim=1).shape == (0, 6, 7, 40)
    with pytest.raises(_lib.CsError, match="overlap"):
        reorder_states(big[:4], p, batch_dim=1, out=big[1:])
    with pytest.raises(_lib.CsError, match="in place"):
        x = torch.zeros(2, 65, 4, device="cuda")
        reorder_states(x, torch.zeros(2, 65, dtype=torch.int64, device="cuda"), out=x)
    with pytest.raises(_lib.CsError, match="adjacent"):
        reorder_states(big, p, batch_dim=1, out=torch.empty_like(rows))
    with pytest.raises(_lib.CsError, match="different devices|no CPU path"):
        reorder_states(big, p.cpu(), batch_dim=1)


def test_states_of_more_than_4_gib():
    B, K, inner = 3, 4, 1 << 20
    outer = 370                                                                          # 4.65 GB
    x = torch.empty(outer, B, K, inner, dtype=torch.uint8, device="cuda")
    tag = torch.arange(outer * B * K, device="cuda").remainder(251).to(torch.uint8).reshape(outer, B, K, 1)
    x.copy_(tag.expand_as(x))
    p = torch.tensor([[1, 0, 3, 3], [0, 1, 2, 3], [3, 2, 1, 0]], device="cuda")
    reorder_states(x, p, batch_dim=1, out=x)
    want = tag[:, torch.arange(B, device="cuda")[:, None], p]
    assert torch.equal(x[..., :1], want) and torch.equal(x[..., -1:], want) and torch.equal(x[..., 12345:12346], want)
    assert bool((x[-1] == want[-1]).all())


def test_logits_and_masks_beyond_4_gib():
    far = (1 << 32) + 12345                                                              # elements between the examples
    big = torch.empty(2 * far, dtype=torch.bfloat16, device="cuda")
    big[:1], big[far:far + 1] = 0, 0
    logits = big.as_strided((2, 3, 3000), (far, 3000, 1))
    g = torch.Generator().manual_seed(6)
    logits.copy_((torch.randn(2, 3, 3000, generator=g) * 2).cuda())
    held = big.view(torch.uint8).as_strided((2, 3, 3000), (2 * far - 4096, 3000, 1), 100000)
    mask = torch.rand(2, 3, 3000, generator=g) < 0.5
    held.copy_(mask)
    check(beam_select(None, logits, 9, mask=held), None, logits.cpu(), 9, mask=mask)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_logits_of_every_magnitude(dtype):
    """The normaliser where the sums of single stretches would leave the range of their type: all logits far below or above
    zero, and stretches of one beam that lie far apart."""
    g = torch.Generator().manual_seed(12)
    x = torch.randn(9, 2, 5000, generator=g) * 2
    for b, shift in enumerate((-689.0, -601.0, -599.0, 599.0, 601.0, 5000.0, -5000.0)):
        x[b] += shift
    x[7, :, :2048] += 900
    x[7, :, 4096:] -= 900
    x[8] *= 300
    logits = x.to(dtype).cuda()
    scores = torch.zeros(9, 2, dtype=torch.float64, device="cuda")
    check(beam_select(scores, logits, 7), scores, logits, 7)
    mask = (torch.rand(9, 1, 5000, generator=g) < 0.3).cuda()
    check(beam_select(scores, logits, 7, mask=mask), scores, logits, 7, mask=mask)


@pytest.mark.parametrize("W", [33, 48, 64])
@pytest.mark.parametrize("B,K,V", [(1, 1, 2048), (2, 40, 64), (1, 3, 6000), (1, 64, 3000), (3, 2, 33000)])
def test_wide_searches(B, K, V, W):
    scores, logits, _ = make(B, K, V, torch.bfloat16, V + W)                             # (many equal values)
    check(beam_select(scores, logits, W), scores, logits, W)
    rows = logits.round()                                                                # (a dozen distinct ones)
    check(beam_select(scores, rows, W), scores, rows, W)


def test_two_hundred_million_values():
    V = 200_000_001
    logits = torch.zeros(1, 1, V, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([V - 1, 0, 123_456_789, 2047, 2048, 99_999_999])
    value = torch.tensor([3.0, 9.0, 5.0, 5.0, 12.0, 0.5])
    logits[0, 0, at.cuda()] = value.bfloat16().cuda()
    lse = float(np.log((V - 6) + np.exp(value.double().numpy()).sum()))
    step = beam_select(torch.zeros(1, 1, dtype=torch.float64, device="cuda"), logits, 8)
    want = [2048, 0, 2047, 123_456_789, V - 1, 99_999_999, 1, 2]      # (then the first of the zeros)
    assert step.tokens[0].tolist() == want and not step.parents.any()
    got = step.scores[0].cpu().numpy() + lse
    assert np.allclose(got, [12.0, 9.0, 5.0, 5.0, 3.0, 0.5, 0.0, 0.0], rtol=0, atol=1e-9)


def test_in_place_with_examples_outermost_in_memory():
    g = torch.Generator().manual_seed(14)
    big = torch.randn(5, 6, 7, 12, generator=g).cuda()
    p = torch.randint(0, 7, (6, 7), generator=g).cuda()
    apart = big.transpose(0, 1).contiguous().transpose(0, 1)
    reorder_states(apart, p, batch_dim=1, out=apart)
    assert torch.equal(apart.cpu(), torch.from_numpy(O.reorder(big.cpu().numpy(), p.cpu().numpy())))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_beams_with_one_value_left_keep_their_score(dtype):
    """A normaliser over one value is that value: the score stays what it was to the last bit, and equal beams keep their
    order."""
    g = torch.Generator().manual_seed(21)
    for B, K, V in ((3, 7, 1), (2, 9, 500), (2, 5, 6000)):
        logits = (torch.randn(B, K, V, generator=g) * 20).to(dtype).cuda()
        keep = torch.randint(0, V, (B, K, 1), generator=g)
        mask = torch.zeros(B, K, V, dtype=torch.bool).scatter_(2, keep, True).cuda()
        for scores in (torch.zeros(B, K, dtype=torch.float64), torch.randn(B, K, generator=g).double().mul(4).round() / 3):
            step = beam_select(scores.cuda(), logits, K, mask=mask)
            order = torch.sort(scores, dim=1, descending=True, stable=True)
            assert torch.equal(step.scores.cpu(), order.values) and torch.equal(step.parents.cpu(), order.indices)
            assert torch.equal(step.tokens.cpu(), keep[:, :, 0].gather(1, order.indices))
    # all but certain beams: what is left of the probability tells them apart
    sure = torch.zeros(1, 6, 3000, dtype=dtype)
    for k, gap in enumerate((24.0, 30.0, 27.0, 33.0, 26.0, 21.0)):
        sure[0, k, :] = -gap
        sure[0, k, 17 * k] = 0.0
    step = beam_select(None, sure.cuda(), 6)
    assert step.parents[0].tolist() == [3, 1, 2, 4, 0, 5]
    want = -np.log1p(2999 * np.exp(-np.array([33.0, 30, 27, 26, 24, 21])))
    assert np.allclose(host(step.scores)[0], want, rtol=1e-4, atol=0)


def test_seventeen_million_examples():
    """More threads than an axis of a launch may hold, in the selection's two kernels and in moving what follows.  The values of
    an example differ by 1/8 and more, so float32 tells them apart."""
    B, K, V = (1 << 24) + 5, 4, 4
    v = torch.arange(B * K, device="cuda").reshape(B, K)
    best = (v * 7 + v // 13) % V
    logits = torch.zeros(B, K, V, dtype=torch.bfloat16, device="cuda")
    logits.scatter_(2, best[..., None], 2.0)
    scores = ((v * 5) % 4).float() * 0.125                                               # of K beams a permutation of 0, 1, 2, 3 eighths
    got = beam_select(scores, logits, 1)
    at = scores.argmax(1, keepdim=True)
    assert torch.equal(got.parents, at)
    assert torch.equal(got.tokens, best.gather(1, at))
    want = 0.375 + 2.0 - math.log(math.exp(2.0) + 3)
    assert float((got.scores.double() - want).abs().max()) <= 2.0 ** -24 * abs(want) + SUM
    del logits, got
    rows = torch.empty(B, 2, 257, dtype=torch.uint8, device="cuda")
    tag = (v[:, :2] * 3 + 1).remainder(251).to(torch.uint8)[..., None]
    rows.copy_(tag.expand_as(rows))
    swap = torch.tensor([1, 0], device="cuda").expand(B, 2)
    moved = reorder_states(rows, swap)
    reorder_states(rows, swap, out=rows)
    assert torch.equal(moved, rows)
    assert bool((rows == tag.flip(1)).all())


@pytest.mark.parametrize("kind", ["plain", "masked", "integers", "far"])
@pytest.mark.parametrize("B,K,V,W", [(700, 1, 2000, 5), (9, 8, 512, 64), (5, 2, 2048, 33), (3, 1, 4096, 64), (1700, 4, 2047, 4),
                                     (100, 8, 100, 64), (40, 3, 1030, 16), (300, 16, 33, 40), (1300, 1, 10200, 40), (1300, 1, 10200, 64),
                                     (6, 13, 900, 7), (520, 2, 9000, 24)])
def test_few_stretches_and_many_examples(B, K, V, W, kind):
    """What one launch does, and what is joined by one wavefront or a few."""
    scores, logits, g = make(B, K, V, torch.float32, B + V + W)
    kw = {}
    if kind == "masked":
        kw = dict(mask=(torch.rand(B, 1, V, generator=g) < 0.4).cuda(), finished=(torch.rand(B, K, generator=g) < 0.3).cuda(),
                  end_token=V // 2)
    elif kind == "integers":      # hundreds of equal values
        logits, scores = logits.round(), scores.round()
        kw = dict(normalise=False)
    elif kind == "far":           # normalisers relative to a stretch's largest value beside absolute ones, in some beams alone
        logits[::3, 0] += 2000
        logits[1::3, :, V // 2:] -= 900
        logits[2::3, -1, : V // 3] = float("-inf")
    check(beam_select(scores, logits, W, **kw), scores, logits, W, **kw)


@pytest.mark.parametrize("K", [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("dtype,inner,skew", [(torch.uint8, 409, 1), (torch.uint8, 16, 3), (torch.uint8, 17, 0), (torch.uint8, 15, 0),
                                              (torch.int16, 205, 1), (torch.int16, 8, 1), (torch.float32, 129, 1), (torch.float32, 64, 1),
                                              (torch.float32, 63, 1), (torch.float32, 66, 2), (torch.float64, 33, 1),
                                              (torch.float64, 34, 0)])
def test_rows_of_every_length_and_alignment(dtype, inner, skew, K):
    """Rows inside wider ones: what lies before and behind them stays."""
    outer, B, pad = 3, 37, skew + 4
    g = torch.Generator().manual_seed(inner + K)
    wide = torch.randint(0, 200, (outer, B, K, inner + pad), generator=g).to(dtype).cuda()
    parents = torch.arange(K).expand(B, K).clone()
    for b in range(B):                                   # from none to all of the chains move, some of them nowhere
        n = b % (K + 1)
        parents[b, torch.randperm(K, generator=g)[:n]] = torch.randint(-1, K + 1, (n,), generator=g)
    fine = (parents >= 0) & (parents < K)
    at = torch.where(fine, parents, torch.arange(K)).cuda()
    want = wide.clone()
    rows = wide[..., skew:skew + inner]
    want[..., skew:skew + inner] = torch.gather(rows, 2, at[None, :, :, None].expand(outer, B, K, inner))
    held = wide.clone()
    target = torch.zeros_like(wide)
    reorder_states(rows, parents.cuda(), batch_dim=1, out=target[..., skew:skew + inner])
    assert torch.equal(target[..., skew:skew + inner], torch.where(fine.cuda()[None, :, :, None], want[..., skew:skew + inner], 0))
    assert not target[..., :skew].any() and not target[..., skew + inner:].any()
    assert torch.equal(wide, held)
    reorder_states(rows, parents.cuda(), batch_dim=1, out=rows)
    assert torch.equal(wide, want)


def test_more_than_four_billion_pieces_of_rows():
    B = 290_000_000
    rows = torch.empty(B, 2, 15, dtype=torch.uint8, device="cuda")
    tag = torch.arange(2 * B, device="cuda").remainder_(251).to(torch.uint8).reshape(B, 2, 1)
    rows.copy_(tag.expand_as(rows))
    swap = torch.tensor([1, 0], device="cuda").expand(B, 2)
    moved = reorder_states(rows, swap)
    assert bool((moved == tag.flip(1)).all())
    del moved
    reorder_states(rows, swap, out=rows)
    assert bool((rows == tag.flip(1)).all())
