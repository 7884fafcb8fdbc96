"""QuantisedHistory against its plain form in float64 (oracle/cs_oracle_beam.py).  Codes are exact, so a value read as
float32 equals code * scale rounded once (2^-24 relative; exact for the power-of-two scales), one read as bfloat16 /
float16 is that rounded once more (2^-8, 2^-11; float16 values below 2^-14 to half of its smallest step, 2^-25)."""
import numpy as np
import pytest
import torch

from oracle import cs_oracle_beam as O
from vae_conditional_sampling_amd import _lib
from vae_conditional_sampling_amd.sampling.beam import beam_select, reorder_states
from vae_conditional_sampling_amd.sampling.utils import QuantisedHistory

pytestmark = pytest.mark.gpu

FORMATS = [("int8", 32), ("int8", 64), ("int8", 128), ("mxfp8", 32), ("mxfp4", 32)]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def close(got, ref, fmt):
    """`ref`: the quantised values in float64."""
    t = got.dtype
    g = got.double().cpu().numpy()
    over = np.abs(ref) > float(torch.finfo(t).max)        # (float16 cannot hold every float32 state)
    assert np.array_equal(np.isnan(g), np.isnan(ref))
    ok = ~np.isnan(ref) & ~over
    tol = (HALF[t] + (2.0 ** -24 if fmt == "int8" else 0)) * np.abs(ref) * (1 + 2.0 ** -7) + TINY[t]
    assert (np.abs(g - ref)[ok] <= tol[ok]).all(), np.abs(g - ref)[ok].max()


def states(shape, g, dtype=torch.float32):
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[-1], generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [1, 2, 7, 8, 9, 21, 31, 32, 33, 43, 64, 65, 127, 129, 784, 1001, 2100])
def test_write_and_read(fmt, group, dtype, D):
    g = torch.Generator().manual_seed(D)
    T, B, K = 5, 3, 2
    q = QuantisedHistory(T, (B, K, D), fmt, group=group)
    assert float(q.read_steps(0, T).abs().max()) == 0.0
    x = states((T, B, K, D), g, dtype)
    q.write(x.cuda(), 2)
    ref = O.quantised(x.double().numpy(), fmt, group)
    close(q.read_steps(2, T), ref, fmt)
    close(q.read_steps(2, T, dtype=dtype), ref, fmt)
    slots = torch.randint(0, T, (4, B, K), generator=g)
    want = ref[(slots.numpy() - 2) % T, np.arange(B)[:, None], np.arange(K)]
    close(q.read(slots.cuda()), want, fmt)
    close(q.read(slots.cuda(), dtype=torch.bfloat16), want, fmt)
    close(q.read(slots[0].cuda()), want[0], fmt)
    chains = torch.randint(0, K, (4, B, 5), generator=g)
    slots = torch.randint(0, T, (4, B, 5), generator=g)
    want = ref[(slots.numpy() - 2) % T, np.arange(B)[:, None], chains.numpy()]
    close(q.read(slots.cuda(), chains.cuda()), want, fmt)


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_every_border_between_two_codes(fmt, group):
    """Values on and one float32 step beside the middle of every two neighbouring codes, at several scales."""
    grid = np.arange(128.0) if fmt == "int8" else np.array(O.E4M3 if fmt == "mxfp8" else O.E2M1)
    mid = ((grid[1:] + grid[:-1]) / 2).astype(np.float32)
    v = np.concatenate([grid.astype(np.float32), mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1e9))])
    v = np.concatenate([v, -v])
    pad = -len(v) % (group - 1)
    v = np.concatenate([v, np.zeros(pad, np.float32)]).reshape(-1, group - 1)
    v = np.concatenate([v, np.full((len(v), 1), grid[-1], np.float32)], axis=1)     # every group holds the largest code
    scales = [1.0, 0.5, 2.0 ** -100, 2.0 ** 100] if fmt != "int8" else [1.0, 2.0 ** -100, 2.0 ** 100, 1.2345, 1 / 3]
    rows = np.concatenate([(v * np.float32(s)).astype(np.float32) for s in scales])
    x = torch.from_numpy(rows)[None, None].permute(2, 0, 1, 3).contiguous()         # [n,1,1,D]
    q = QuantisedHistory(x.shape[0], (1, 1, group), fmt, group=group)
    q.write(x.cuda(), 0)
    ref = O.quantised(rows, fmt, group)
    close(q.read_steps(0, x.shape[0])[:, 0, 0], ref, fmt)
    if fmt != "int8":
        assert np.array_equal(q.read_steps(0, x.shape[0])[:, 0, 0].double().cpu().numpy(), ref)


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_integers_of_random_scales_round_to_the_nearest(fmt, group):
    """Many quotients near a border: random multiples of half a scale, each moved by a few float32 steps."""
    g = np.random.RandomState(group)
    n = 2000
    top = np.exp2(g.uniform(-20, 20, (n, 1))).astype(np.float32)
    s = (top / np.float32(127)).astype(np.float64)
    x = ((g.randint(-253, 254, (n, group)) / 2) * s).astype(np.float32)
    x = np.where(x != 0, (x.view(np.int32) + g.randint(-2, 3, x.shape).astype(np.int32)).view(np.float32), x)
    x = np.clip(x, -top, top)
    x[:, :1] = top
    t = torch.from_numpy(x).reshape(n, 1, 1, group)
    q = QuantisedHistory(n, (1, 1, group), fmt, group=group)
    q.write(t.cuda(), 0)
    close(q.read_steps(0, n)[:, 0, 0], O.quantised(x, fmt, group), fmt)


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_the_largest_of_a_group_chooses_its_scale(fmt, group):
    """Largest magnitudes on, below and above the end of the elements' range and of powers of two."""
    ends = np.float32([448.0, 6.0, 127.0, 1.0, 256.0, 0.75, 0.875, 3.0])
    tops = np.concatenate([ends, np.nextafter(ends, np.float32(0)), np.nextafter(ends, np.float32(1e9))])
    tops = np.concatenate([(tops * np.float32(s)).astype(np.float32) for s in (1.0, 2.0 ** -60, 2.0 ** 70, 2.0 ** -120)])
    x = np.random.RandomState(1).uniform(-1, 1, (len(tops), group)).astype(np.float32) * tops[:, None]
    x[:, 5] = -tops
    t = torch.from_numpy(x).reshape(len(tops), 1, 1, group)
    q = QuantisedHistory(len(tops), (1, 1, group), fmt, group=group)
    q.write(t.cuda(), 0)
    close(q.read_steps(0, len(tops))[:, 0, 0], O.quantised(x, fmt, group), fmt)


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_zeros_tiny_huge_and_not_finite_values(fmt, group):
    inf, nan, f = float("inf"), float("nan"), torch.finfo(torch.float32)
    D = 2 * group + 5
    x = torch.zeros(12, 1, 1, D)
    x[1] = 1e-42                                     # denormal
    x[2, ..., 0] = f.tiny
    x[3] = f.max
    x[3, ..., 1::2] = -f.max
    x[4, ..., 3] = f.min                             # the lowest value beside ordinary ones
    x[4, ..., 0] = 1.0
    x[5] = torch.randn(D, generator=torch.Generator().manual_seed(0))
    x[5, ..., group] = nan                           # one group holds NaN, the others not
    x[6] = x[5].nan_to_num(0.5)
    x[6, ..., 2], x[6, ..., 3] = inf, -inf
    x[7] = nan
    x[8] = -inf
    x[9] = -0.0
    x[10, ..., -1] = 3.0                             # the last group, a part of one
    x[11] = 2.0 ** -140
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        y[3] = y[3].clamp(torch.finfo(dtype).min, torch.finfo(dtype).max)
        q = QuantisedHistory(12, (1, 1, D), fmt, group=group)
        q.write(y.cuda(), 0)
        close(q.read_steps(0, 12), O.quantised(y.double().numpy(), fmt, group), fmt)


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_ragged_writes_leave_all_else_as_it_was(fmt, group):
    g = torch.Generator().manual_seed(8)
    T, B, K, D, n = 7, 4, 3, 43, 5
    q = QuantisedHistory(T, (B, K, D), fmt, group=group)
    q.data.copy_(torch.randint(0, 256, q.data.shape, generator=g).to(torch.uint8))      # (whatever it held)
    before = q.data.clone()
    x = states((n, B, K, D), g)
    start = torch.randint(0, 3 * T, (B, K), generator=g)
    start[0, 1], start[2, 2] = -1, -(1 << 40)
    start[1, 0] = (1 << 40) * T + 3                                                       # a far position
    counts = torch.randint(0, n + 1, (B, K), generator=g)
    counts[0, 0], counts[0, 2], counts[3, 0], counts[1, 0] = 0, n + 100, -3, n
    q.write(x.cuda(), start.cuda(), counts.cuda())
    ref = O.quantised(x.numpy(), fmt, group)
    touched = torch.zeros(T, B, K, dtype=torch.bool)
    for b in range(B):
        for k in range(K):
            for i in range(min(max(int(counts[b, k]), 0), n)):
                if start[b, k] >= 0:
                    s = (int(start[b, k]) + i) % T
                    touched[s, b, k] = True
                    got = q.read(torch.full((B, K), s).cuda())[b, k]
                    close(got, ref[i, b, k], fmt)
    assert 10 < int(touched.sum()) < T * B * K
    assert torch.equal(q.data.cpu()[~touched], before.cpu()[~touched])


def test_slots_and_chains_that_do_not_exist_read_as_zeros():
    g = torch.Generator().manual_seed(4)
    q = QuantisedHistory(3, (2, 2, 33), "mxfp8")
    q.write(states((3, 2, 2, 33), g).cuda(), 0)
    slots = torch.tensor([[[0, -1], [3, 2]], [[1 << 40, 1], [-5, 0]]]).cuda()
    out = q.read(slots)
    fine = (slots >= 0) & (slots < 3)
    assert bool((out[~fine] == 0).all()) and bool((out[fine] != 0).any(dim=-1).all())
    chains = torch.tensor([[[0, 2], [1, -1]], [[0, 1], [1 << 33, 0]]]).cuda()
    out = q.read(torch.zeros_like(slots), chains)
    fine = (chains >= 0) & (chains < 2)
    assert bool((out[~fine] == 0).all()) and bool((out[fine] != 0).any(dim=-1).all())


def test_strides_and_windows():
    g = torch.Generator().manual_seed(6)
    T, B, K, D = 6, 3, 4, 43
    x = states((2 * T, B, K, 50), g).cuda()
    view = x[::2, :, :, 3:46]                        # rows of 50, every other step
    q, p = QuantisedHistory(T, (B, K, D), "int8"), QuantisedHistory(T, (B, K, D), "int8")
    q.write(view, 0)
    p.write(view.contiguous(), 0)
    assert torch.equal(q.data, p.data)
    q.write(x[0, :, :, 7:50], 3)                     # one step, [B,K,D]
    p.write(x[0, :, :, 7:50].contiguous()[None], 3)
    assert torch.equal(q.data, p.data)
    q.write(view[0, :1, :1].expand(B, K, D), 4)      # one state for all
    p.write(view[0, :1, :1].expand(B, K, D).contiguous(), 4)
    assert torch.equal(q.data, p.data)
    q.write(view.half().transpose(1, 2).contiguous().transpose(1, 2), 1)
    p.write(view.half().contiguous(), 1)
    assert torch.equal(q.data, p.data)
    slots = torch.randint(0, T, (5, B, K), generator=g).cuda()
    ref = q.read(slots)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        wide = torch.full((5, B, K + 2, D + 3), 7.0, dtype=dtype, device="cuda")
        q.read(slots, out=wide[:, :, 1:K + 1, 2:D + 2])
        assert torch.equal(wide[:, :, 1:K + 1, 2:D + 2], ref.to(dtype))
        wide[:, :, 1:K + 1, 2:D + 2] = 7.0
        assert bool((wide == 7.0).all())             # nothing around the window
    with pytest.raises(_lib.CsError, match="place of its own"):
        q.read(slots, out=torch.zeros(1, B, K, D, device="cuda").expand(5, B, K, D))
    assert torch.equal(q.read_steps(4, 9), q.read(((4 + torch.arange(9)) % T)[:, None, None].expand(9, B, K).cuda()))
    assert q.read(slots[:0]).shape == (0, B, K, D)
    empty = QuantisedHistory(3, (0, 2, 5), "mxfp4")
    empty.write(torch.zeros(2, 0, 2, 5, device="cuda"), 0)
    assert empty.read_steps(0, 2).shape == (2, 0, 2, 5)


def test_ring_of_more_than_4_gib():
    T, B, K, D = 300, 2, 2, 1 << 22                  # 300 x 4 records of 4 MiB + scales: 5.2 GB
    q = QuantisedHistory(T, (B, K, D), "mxfp8")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, B, K, D, generator=g, device="cuda").bfloat16()
    q.write(x, T - 1)                                # the last slot and the first
    back = q.read_steps(T - 1, 2, dtype=torch.bfloat16)
    small = QuantisedHistory(2, (B, K, D), "mxfp8")
    small.write(x, 0)
    assert torch.equal(back, small.read_steps(0, 2, dtype=torch.bfloat16))
    assert float((back.float() - x.float()).abs().max()) <= 2.0 ** -4 * float(x.float().abs().max())
    assert float(q.read_steps(1, 1).abs().max()) == 0.0
    q.reorder(torch.tensor([[1, 0], [1, 1]], device="cuda"))
    assert torch.equal(q.read_steps(T - 1, 1, dtype=torch.bfloat16)[0, 0, 0], back[0, 0, 1])


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_reorder_moves_whole_states(fmt, group):
    g = torch.Generator().manual_seed(2)
    T, B, K, D = 5, 4, 6, 70
    q = QuantisedHistory(T, (B, K, D), fmt, group=group)
    q.write(states((T, B, K, D), g).cuda(), 0)
    before = q.read_steps(0, T)
    p = torch.randint(0, K, (B, K), generator=g).cuda()
    q.reorder(p, steps=3)
    after = q.read_steps(0, T)
    assert torch.equal(after[3:], before[3:])
    assert torch.equal(after[:3], before[:3][:, torch.arange(B, device="cuda")[:, None], p])


def _search(fmt, group, steps, B, K, V, D, seed, *, own):
    """A beam search whose states are kept quantised: the state of a step is half the kept state of the step before plus
    the chosen value's vector, its logits a projection of it.  Plain: numpy in float64 (products of few exact values are
    made exact by integers: states and tables hold multiples of 2^-6)."""
    g = torch.Generator().manual_seed(seed)
    table = torch.randint(-64, 65, (V, D), generator=g).float() / 64
    proj = torch.randint(-4, 5, (D, V), generator=g).float() / 4
    end = 1
    state = torch.zeros(B, K, D)
    if own:
        q = QuantisedHistory(steps, (B, K, D), fmt, group=group)
        scores = torch.full((B, K), float("-inf"), dtype=torch.float64)
        scores[:, 0] = 0
        scores, table, proj, state = scores.cuda(), table.cuda(), proj.cuda(), state.cuda()
        finished = torch.zeros(B, K, dtype=torch.bool, device="cuda")
        drawn = torch.zeros(B, K, steps, dtype=torch.int64, device="cuda")
        for t in range(steps):
            q.write(state, t)
            logits = (state.double() @ proj.double()).float()
            scores, parents, tokens = beam_select(scores, logits, K, finished=finished, end_token=end)
            q.reorder(parents, steps=t + 1)
            drawn = reorder_states(drawn, parents)
            drawn[:, :, t] = tokens
            finished = finished.gather(1, parents) | (tokens == end)
            kept = q.read_steps(t, 1)[0]
            state = 0.5 * kept + table[tokens]
        return scores.cpu().numpy(), drawn.cpu().numpy(), q.read_steps(0, steps).double().cpu().numpy()
    scores = np.full((B, K), -np.inf)
    scores[:, 0] = 0
    table, proj, state = table.numpy().astype(np.float64), proj.numpy().astype(np.float64), state.numpy().astype(np.float64)
    ring = np.zeros((steps, B, K, D))
    finished = np.zeros((B, K), bool)
    drawn = np.zeros((B, K, steps), np.int64)
    for t in range(steps):
        ring[t] = O.quantised(state.astype(np.float32), fmt, group).astype(np.float32)
        logits = (state @ proj).astype(np.float32)
        scores, parents, tokens = O.beam_select(scores, logits, K, finished=finished, end_token=end)
        ring[:t + 1] = O.reorder(ring[:t + 1], parents)
        drawn = O.reorder(drawn[None], parents)[0]
        drawn[:, :, t] = tokens
        finished = np.take_along_axis(finished, parents, 1) | (tokens == end)
        state = (np.float32(0.5) * ring[t].astype(np.float32) + table[tokens].astype(np.float32)).astype(np.float64)
    return scores, drawn, ring


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("B,K,V,D", [(1, 1, 20, 16), (3, 4, 300, 43), (2, 6, 2500, 33)])
def test_a_search_over_a_quantised_history(fmt, group, B, K, V, D):
    own = _search(fmt, group, 12, B, K, V, D, 3, own=True)
    plain = _search(fmt, group, 12, B, K, V, D, 3, own=False)
    assert np.array_equal(own[1], plain[1])
    assert np.allclose(own[0], plain[0], rtol=1e-12, atol=1e-9)
    assert np.array_equal(own[2], plain[2])


def test_captured_step_replays_with_new_inputs():
    """write, select, reorder and read in one graph, replayed between eager work on the same tensors' successors."""
    g = torch.Generator().manual_seed(11)
    T, B, K, D, V = 6, 3, 4, 43, 5000
    x = torch.zeros(B, K, D, device="cuda")
    logits = torch.zeros(B, K, V, device="cuda", dtype=torch.bfloat16)
    scores = torch.zeros(B, K, device="cuda")
    start = torch.zeros(B, K, dtype=torch.int64, device="cuda")
    slots = torch.zeros(2, B, K, dtype=torch.int64, device="cuda")
    q, e = QuantisedHistory(T, (B, K, D), "int8"), QuantisedHistory(T, (B, K, D), "int8")

    def step(h, x, logits, scores, start, slots):
        h.write(x, start)
        s = beam_select(scores, logits, K)
        h.reorder(s.parents)
        return (*s, reorder_states(x, s.parents), h.read(slots))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step(q, x, logits, scores, start, slots)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, x, logits, scores, start, slots)
    q.data.zero_()
    for i in range(4):
        x.copy_(torch.randn(B, K, D, generator=g))
        logits.copy_(torch.randn(B, K, V, generator=g))
        scores.copy_(torch.randn(B, K, generator=g))
        start.copy_(torch.randint(0, T, (B, K), generator=g))
        slots.copy_(torch.randint(0, T, (2, B, K), generator=g))
        graph.replay()
        ref = step(e, x.clone(), logits.clone(), scores.clone(), start.clone(), slots.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
        assert torch.equal(q.data, e.data)


def test_a_billion_states_in_one_call():
    """More threads than an axis of a launch may hold.  Integers up to 100 beside a value of 127 have a scale of one in int8."""
    B, K, D = 1 << 20, 1025, 2
    q = QuantisedHistory(1, (B, K, D), "int8", group=32)
    x = torch.full((B, K, D), 127, dtype=torch.float16, device="cuda")
    x[..., 1] = (torch.arange(B * K, device="cuda") % 101).reshape(B, K)
    q.write(x, 0)
    back = q.read_steps(0, 1, dtype=torch.float16)
    assert torch.equal(back[0], x)
    at = torch.zeros(1, 1, 1, dtype=torch.int64, device="cuda").expand(1, B, K)
    back.zero_()
    assert torch.equal(q.read(at, out=back)[0], x)
