"""GPU parity of the channels-last group norm against the 64-bit oracle.

Tolerance, with U = 2^-24 and everything in units of the group's deviation. Rounding after the
statistics: the deviation from the mean, the scale w / deviation, the remainder of the bias and the
multiply-add round under 6 U (|z| + |b|) together. Statistics: a column's differences from its first
value of up to 32 rows, |d| <= D, are summed in fp32. The differences round by U D, and the k-th of m
additions by U k D, so a run's sum is off by at most U D (m + m (m + 1) / 2) and its mean by
U D (1 + (m + 1) / 2) <= 18 U D (m = 32); of the squares likewise, the difference's rounding counting
twice and the product's once: the mean square by U D^2 (3 + (m + 1) / 2) <= 20 U D^2. (All above the
runs is fp64.) The shift by the run's reference moves the mean's error R into the mean square by 2 R D.
So the mean is off by 18 U D and the variance by 56 U D^2, 1 / sqrt(var) by half that, relative:
|dz| <= |w| 18 U D + (|z| + |b|) 28 U D^2, D <= twice the largest |x - mean| of window and group. (Rounding
errors have either sign; the sums' true error is far below.) ReLU and SiLU pass an error on with a
slope of at most 1.1, SiLU adds under 8 U of its result; then half a step of the output's type.
"""
import numpy as np
import pytest
import torch

from oracle import int8 as oi
from parakeet_cuda_b200 import pq8
from parakeet_cuda_b200.pq8 import EPI_NONE, EPI_RELU, EPI_RESIDUAL, EPI_SILU, FLAG_OUT_TF32
from parakeet_cuda_b200.runtime import Int8Weight, Runtime

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)
ACTS = {'none': EPI_NONE, 'relu': EPI_RELU, 'silu': EPI_SILU}
U = 2.0 ** -24


@pytest.fixture(scope='module')
def rt():
    return Runtime(0)


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def f64(t):
    return t.double().cpu().numpy()


def inputs(seed, rows, channels, dtype, offset=0.5):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(rows, channels)) * np.exp(0.5 * rng.normal(size=(1, channels))) + offset
    w, b = 1 + 0.2 * rng.normal(size=channels), 0.2 * rng.normal(size=channels)
    return dev(x.astype(np.float32), dtype), dev(w.astype(np.float32)), dev(b.astype(np.float32))


def spread(x, groups, bounds):
    """D of the module's tolerance for every value: twice the largest |x - mean| / sqrt(var + eps)."""
    c = x.shape[1]
    one, zero = np.ones(c), np.zeros(c)
    z = np.abs(oi.group_norm(x, one, zero, groups, bounds))
    out = np.zeros_like(z)
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        if hi > lo:
            blk = z[lo:hi].reshape(hi - lo, groups, c // groups)
            out[lo:hi] = (0 * blk + 2 * blk.max(axis=(0, 2), keepdims=True)).reshape(hi - lo, c)
    return out


def check(got, x, w, b, groups, bounds, act, extra=0.0):
    z = oi.group_norm(f64(x), f64(w), f64(b), groups, bounds)
    far = spread(f64(x), groups, bounds)
    y = oi.act(z, act)
    inside = np.zeros(len(z), bool)
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        inside[lo:hi] = True
    g, y, z, far = f64(got)[inside], y[inside], z[inside], far[inside]
    size = np.abs(z) + np.abs(f64(b))
    err = 1.1 * U * (6 * size + 18 * far * np.abs(f64(w)) + 28 * far ** 2 * size) + 8 * U * np.abs(y)
    fi = torch.finfo(got.dtype)
    bound = err + fi.eps / 2 * (np.abs(y) + err) + fi.tiny * fi.eps + extra * np.abs(y) + 1e-37
    assert np.isfinite(g).all()
    bad = np.abs(g - y) > bound
    assert not bad.any(), (int(bad.sum()), float((np.abs(g - y) / bound).max()))


# one row, one channel per group, odd groups and channels, one group over everything, long windows
SHAPES = [(1, 1, 4, 4), (1, 1, 32, 1), (3, 7, 1024, 32), (2, 50, 96, 96), (1, 333, 1000, 8), (4, 17, 35, 5), (2, 1, 2048, 1),
          (1, 3000, 64, 1), (8, 375, 1024, 32), (1, 900, 1024, 1), (2, 130, 4096, 2), (1, 40, 16384, 4096), (70, 3, 16, 2),
          (1, 2000, 24, 3)]


@pytest.mark.parametrize('windows,t,channels,groups', SHAPES)
@pytest.mark.parametrize('dtype', TYPES)
def test_group_norm(rt, windows, t, channels, groups, dtype):
    x, w, b = inputs(windows + t, windows * t, channels, dtype)
    act = list(ACTS)[(t + channels) % 3]
    y = rt.group_norm(x, w, b, groups, windows=windows, epilogue=ACTS[act])
    check(y, x, w, b, groups, [i * t for i in range(windows + 1)], act)


RAGGED = [[0, 0, 1, 5, 5, 300, 301, 640], [3, 10, 200, 600], [0, 640], [640, 640], [100, 100, 101]]


@pytest.mark.parametrize('bounds', RAGGED)
@pytest.mark.parametrize('channels,groups', [(256, 8), (1000, 8), (1024, 1)])
def test_group_norm_ragged(rt, bounds, channels, groups):
    """Empty windows, one-row windows, rows before the first window and behind the last: those keep their bytes."""
    for dtype in TYPES:
        x, w, b = inputs(len(bounds), 640, channels, dtype)
        out = torch.full_like(x, 9.0)
        off = torch.tensor(bounds, dtype=torch.int32, device='cuda')
        rt.group_norm(x, w, b, groups, windows=len(bounds) - 1, offsets=off, epilogue=EPI_SILU, out=out)
        check(out, x, w, b, groups, bounds, 'silu')
        assert (out[:bounds[0]] == 9).all() and (out[bounds[-1]:] == 9).all()


def test_group_norm_rows_outside_do_not_matter(rt):
    """NaN and infinities in rows of no window change nothing; in a window they stay in its group."""
    x, w, b = inputs(5, 64, 64, torch.float32)
    off = torch.tensor([8, 20, 50], dtype=torch.int32, device='cuda')
    clean = rt.group_norm(x, w, b, 4, windows=2, offsets=off)
    x2 = x.clone()
    x2[:8], x2[50:] = float('nan'), float('inf')
    assert torch.equal(rt.group_norm(x2, w, b, 4, windows=2, offsets=off)[8:50], clean[8:50])
    x2[30, 20] = float('nan')  # window 1, group 1
    got = rt.group_norm(x2, w, b, 4, windows=2, offsets=off)
    assert torch.isnan(got[20:50, 16:32]).all()
    assert torch.equal(got[8:20], clean[8:20])
    assert torch.equal(got[20:50, :16], clean[20:50, :16]) and torch.equal(got[20:50, 32:], clean[20:50, 32:])


def test_group_norm_offsets_outside_the_rows(rt):
    """Offsets beyond the rows are held inside; falling ones leave the values of their rows open, but nothing
    outside the output is touched."""
    for channels, groups in ((64, 4), (1000, 8), (35, 5)):  # one launch, units that straddle groups, single columns
        x, w, b = inputs(6, 32, channels, torch.float32)
        guard = torch.full((3, 32, channels), 5.0, device='cuda')
        off = torch.tensor([-7, 10, 10, 1000, 2 ** 31 - 1], dtype=torch.int32, device='cuda')
        rt.group_norm(x, w, b, groups, windows=4, offsets=off, out=guard[1])
        check(guard[1], x, w, b, groups, [0, 10, 10, 32], 'none')
        for bad in ([20, 10, 4, 1000, -5], [2 ** 31 - 1, 0, 32, 16, 31], [-2 ** 31, -1, 40, 3, 3]):
            rt.group_norm(x, w, b, groups, windows=4, out=guard[1],
                          offsets=torch.tensor(bad, dtype=torch.int32, device='cuda'))
            if channels % 16 == 0:
                rt.group_norm_quantize(x, w, b, groups, windows=4,
                                       offsets=torch.tensor(bad, dtype=torch.int32, device='cuda'))
        assert (guard[0] == 5).all() and (guard[2] == 5).all()


def test_group_norm_large_offset_and_long_window(rt):
    """A common offset of 10^4 deviations, and 40,000 rows in one window: statistics keep their digits."""
    x, w, b = inputs(7, 1000, 64, torch.float32, offset=1e4)
    check(rt.group_norm(x, w, b, 4), x, w, b, 4, [0, 1000], 'none')
    x, w, b = inputs(8, 40000, 32, torch.float16, offset=0.0)
    check(rt.group_norm(x, w, b, 2), x, w, b, 2, [0, 40000], 'none')
    x[:] = 3.25  # no variance at all
    y = rt.group_norm(x, w, b, 2)
    assert torch.equal(y, b.to(torch.float16).expand_as(y))


def test_group_norm_misaligned_and_tf32(rt):
    flat = torch.randn(65 * 64 + 3, device='cuda')
    w, b = torch.ones(64, device='cuda'), torch.zeros(64, device='cuda')
    for skip in (0, 1, 3):
        x = flat[skip:skip + 65 * 64].view(65, 64)
        check(rt.group_norm(x, w, b, 4), x, w, b, 4, [0, 65], 'none')
        got = rt.group_norm(x, w, b, 4, flags=FLAG_OUT_TF32)
        bits = got.view(torch.int32)
        assert not (bits & 0x1FFF).any()
        check(got, x, w, b, 4, [0, 65], 'none', extra=2.0 ** -11)
        h = flat.half()[skip:skip + 65 * 64].view(65, 64)
        check(rt.group_norm(h, w, b, 4), h, w, b, 4, [0, 65], 'none')


@pytest.mark.parametrize('windows,t,channels,groups', [(3, 7, 1024, 32), (1, 100, 48, 3), (2, 30, 1040, 1), (5, 9, 2048, 16),
                                                       (1, 4, 16384, 4096), (8, 40, 640, 40)])
@pytest.mark.parametrize('dtype', TYPES)
def test_group_norm_quantize(rt, windows, t, channels, groups, dtype):
    """The oracle's scales and integers, but for values within 1e-9 of a border (fp64 on both sides)."""
    for act in ACTS:
        x, w, b = inputs(windows * t, windows * t, channels, dtype)
        got = rt.group_norm_quantize(x, w, b, groups, windows=windows, epilogue=ACTS[act])
        h = oi.group_norm(f64(x), f64(w), f64(b), groups, [i * t for i in range(windows + 1)], epilogue=act)
        q, s, margin = oi.quantize(h)
        gs = got.scale.cpu().numpy()
        assert (np.abs(gs - s) <= 2.0 ** -23 * s).all() and (gs == s).mean() >= 0.99
        wrong = got.q.cpu().numpy() != q
        assert not (wrong & (margin > 1e-9)[...] & (gs == s)[:, None]).any(), int(wrong.sum())


def test_conv_module_tail(rt):
    """Group norm + SiLU quantised, then the 8-bit pointwise_conv2 with the residual, over ragged windows: as the
    oracle's chain, within the product's bound. Rows of no window keep the residual stream they had."""
    rng = np.random.default_rng(12)
    bounds = [0, 40, 40, 155, 260]
    off = torch.tensor(bounds, dtype=torch.int32, device='cuda')
    x, w, b = inputs(13, 260, 1024, torch.float32)
    wq, t = rng.integers(-127, 128, size=(1024, 1024)).astype(np.int8), (rng.uniform(.5, 2, 1024) * 1e-3).astype(np.float32)
    resid = dev(rng.normal(size=(260, 1024)).astype(np.float32))

    def step():
        h = rt.group_norm_quantize(x, w, b, 32, windows=4, offsets=off, epilogue=EPI_SILU)
        return rt.linear_i8(h, Int8Weight(dev(wq), dev(t)), resid=resid, epilogue=EPI_RESIDUAL)

    got = step()
    q, s, margin = oi.quantize(oi.group_norm(f64(x), f64(w), f64(b), 32, bounds, epilogue='silu'))
    assert margin.min() > 1e-9
    z, size = oi.product(q, s, wq, t)
    y = f64(resid) + z
    assert (np.abs(f64(got) - y) <= 5 * U * size + 2 * U * np.abs(y)).all()
    assert torch.equal(step(), got)
    assert rt.device_status() == 0


def test_group_norm_graph_and_streams(rt):
    x, w, b = inputs(14, 8 * 60, 512, torch.bfloat16)
    want = rt.group_norm(x, w, b, 16, windows=8, epilogue=EPI_SILU)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rt.group_norm(x, w, b, 16, windows=8, epilogue=EPI_SILU)
        quant = rt.group_norm_quantize(x, w, b, 16, windows=8, epilogue=EPI_SILU)
    out.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    again = rt.group_norm_quantize(x, w, b, 16, windows=8, epilogue=EPI_SILU)
    assert torch.equal(again.q, quant.q) and torch.equal(again.scale, quant.scale)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(rt.group_norm(x, w, b, 16, windows=8, epilogue=EPI_SILU))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_group_norm_refuses(rt):
    x, w, b = torch.zeros(12, 64, device='cuda'), torch.ones(64, device='cuda'), torch.zeros(64, device='cuda')
    off = torch.tensor([0, 6, 12], dtype=torch.int32, device='cuda')
    bad = [lambda: rt.group_norm(x.double(), w, b, 4), lambda: rt.group_norm(x.cpu(), w, b, 4),
           lambda: rt.group_norm(x[:, ::2], w[:32], b[:32], 4), lambda: rt.group_norm(x, w[:32], b, 4),
           lambda: rt.group_norm(x, w.half(), b, 4), lambda: rt.group_norm(x, w, b, 4, windows=5),
           lambda: rt.group_norm(x, w, b, 4, windows=0), lambda: rt.group_norm(x, w, b, 4, windows=3, offsets=off),
           lambda: rt.group_norm(x, w, b, 4, windows=2, offsets=off.long()),
           lambda: rt.group_norm(x, w, b, 4, windows=2, offsets=off.cpu()),
           lambda: rt.group_norm(x, w, b, 4, out=torch.zeros(12, 32, device='cuda')),
           lambda: rt.group_norm(x, w, b, 4, out=torch.zeros(12, 64, device='cuda', dtype=torch.float16)),
           lambda: rt.group_norm(x.view(3, 4, 64), w, b, 4)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    for f in (lambda: rt.group_norm(x, w, b, 5), lambda: rt.group_norm(x, w, b, 4, out=x),
              lambda: rt.group_norm(x, w, b, 4, epilogue=EPI_RESIDUAL), lambda: rt.group_norm(x, w, b, 4, eps=0.0),
              lambda: rt.group_norm(x.half(), w, b, 4, flags=FLAG_OUT_TF32),
              lambda: rt.group_norm_quantize(torch.zeros(4, 24, device='cuda'), w[:24], b[:24], 2)):
        with pytest.raises(pq8.PQ8Error):
            f()
    assert rt.group_norm(x[:0], w, b, 4).shape == (0, 64)


def test_group_norm_bad_values_pass_every_activation(rt):
    """An infinity or a NaN makes its group NaN through every activation; values too far apart for squares in
    fp32 give NaN or the right result; other groups and windows keep their bits. Quantised, a bad value takes its rows' scales."""
    for channels, groups, dtype in ((64, 4, torch.float32), (1000, 8, torch.float16), (35, 5, torch.float32)):
        x, w, b = inputs(15, 60, channels, dtype)
        cg = channels // groups
        values = [float('inf'), float('nan')] + ([3e38, 1e30] if dtype == torch.float32 else [])
        for name, act in ACTS.items():
            clean = rt.group_norm(x, w, b, groups, windows=3, epilogue=act)
            for value in values:
                y = x.clone()
                y[25, cg + 1] = value  # window 1, group 1
                got = rt.group_norm(y, w, b, groups, windows=3, epilogue=act)
                nan = torch.isnan(got[20:40, cg:2 * cg])
                assert nan.all() if not np.isfinite(value) else nan.all() or not nan.any(), (channels, act, value)
                if not nan.any():
                    check(got, y, w, b, groups, [0, 20, 40, 60], name)
                got[20:40, cg:2 * cg] = clean[20:40, cg:2 * cg]
                assert torch.equal(got, clean)
    x, w, b = inputs(16, 60, 64, torch.float32)
    for act in ACTS.values():
        clean = rt.group_norm_quantize(x, w, b, 4, windows=3, epilogue=act)
        for value in (float('inf'), float('nan')):
            y = x.clone()
            y[25, 17] = value
            got = rt.group_norm_quantize(y, w, b, 4, windows=3, epilogue=act)
            assert torch.isnan(got.scale[20:40]).all() and not got.q[20:40].any()
            assert torch.equal(got.scale[:20], clean.scale[:20]) and torch.equal(got.q[40:], clean.q[40:])


def test_group_norm_refuses_sizes(rt):
    x, w, b = torch.zeros(12, 64, device='cuda'), torch.ones(64, device='cuda'), torch.zeros(64, device='cuda')
    for groups in (0, -4, 128, (1 << 32) + 4):
        with pytest.raises(ValueError):
            rt.group_norm(x, w, b, groups)
    with pytest.raises(ValueError):
        rt.group_norm(x[:0], w, b, 4, windows=1 << 32)


def test_group_norm_past_32_bit_offsets(rt):
    """More than 2^31 values, windows of equal and of unequal lengths: the last window is right."""
    torch.manual_seed(17)
    channels, t = 1024, 3000
    windows = (1 << 31) // (channels * t) + 2
    x = torch.randn(windows * t, channels, device='cuda', dtype=torch.bfloat16)
    _, w, b = inputs(17, 1, channels, torch.float32)
    last = x[(windows - 1) * t:].clone()
    for groups in (32, 1):  # one launch, two launches
        y = rt.group_norm(x, w, b, groups, windows=windows, epilogue=EPI_SILU)
        check(y[(windows - 1) * t:], last, w, b, groups, [0, t], 'silu')
        off = torch.tensor([0, 5, windows * t - 77, windows * t], dtype=torch.int32, device='cuda')
        rt.group_norm(x, w, b, groups, windows=3, offsets=off, epilogue=EPI_SILU, out=y)
        check(y[-77:], x[-77:], w, b, groups, [0, 77], 'silu')
    del y
    got = rt.group_norm_quantize(x, w, b, 32, windows=windows, epilogue=EPI_SILU)
    alone = rt.group_norm_quantize(last, w, b, 32, epilogue=EPI_SILU)
    assert torch.equal(got.scale[(windows - 1) * t:], alone.scale) and torch.equal(got.q[(windows - 1) * t:], alone.q)
