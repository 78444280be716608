"""The group norm's windows and groups at their edges: windows that leave rows out, many windows, groups wider than a
CTA. The oracle and the tolerances of the quantised form are those of test_gpu_group_norm.py: integers equal but for
values within 1e-9 of a border, scales within one step of fp32."""
import numpy as np
import pytest
import torch

from oracle import int8 as oi
from parakeet_cuda_b200.pq8 import EPI_RESIDUAL, EPI_SILU
from parakeet_cuda_b200.runtime import ELEMENT_TYPES, Int8Weight, Runtime

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)


@pytest.fixture(scope='module')
def rt():
    return Runtime(0)


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def f64(t):
    return t.double().cpu().numpy()


def inputs(seed, rows, channels, dtype, skip=0):
    rng = np.random.default_rng(seed)
    flat = dev(rng.normal(size=rows * channels + skip).astype(np.float32) + 0.5, dtype)
    w, b = 1 + 0.2 * rng.normal(size=channels), 0.2 * rng.normal(size=channels)
    return flat[skip:].view(rows, channels), dev(w.astype(np.float32)), dev(b.astype(np.float32))


def check_quantized(q, scale, x, w, b, groups, bounds, act):
    h = oi.group_norm(f64(x), f64(w), f64(b), groups, bounds, epilogue=act)
    inside = np.zeros(len(h), bool)
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        inside[lo:hi] = True
    wq, ws, margin = oi.quantize(h[inside])
    q, scale = q.cpu().numpy(), scale.cpu().numpy()
    assert (np.abs(scale[inside] - ws) <= 2.0 ** -23 * ws).all()
    wrong = q[inside] != wq
    assert not (wrong & (margin > 1e-9) & (scale[inside] == ws)[:, None]).any(), int(wrong.sum())
    assert not q[~inside].any() and (scale[~inside] == 0).all()


# rows left out before, behind and (by offsets that start past 0) around one window; empty windows at both ends; none
BOUNDS = [[0, 0, 0, 7, 90, 90, 200, 200], [13, 20, 64, 187], [60, 140], [100, 100], [200, 200, 200], [0]]


@pytest.mark.parametrize('bounds', BOUNDS)
@pytest.mark.parametrize('channels,groups,skip', [(64, 4, 0), (1024, 32, 0), (1040, 8, 0), (64, 4, 1), (9008, 1, 0)])
def test_quantize_leaves_rows_out(rt, bounds, channels, groups, skip):
    """Rows of no window are zeros with scale 0, whatever the buffers held, in every kernel form."""
    rows, windows = 200, len(bounds) - 1
    off = torch.tensor(bounds, dtype=torch.int32, device='cuda')
    for dtype in TYPES:
        x, w, b = inputs(channels + windows, rows, channels, dtype, skip)
        q = torch.full((rows + 2, channels), 77, dtype=torch.int8, device='cuda')
        scale = torch.full((rows + 2,), float('nan'), device='cuda')
        kind = ELEMENT_TYPES[dtype]
        need = rt.lib.group_norm_workspace_size(kind, rows, windows, channels, groups, True, True, skip == 0)
        ws = torch.empty(need, dtype=torch.uint8, device='cuda')
        rt.lib.call('pq8_group_norm_quantize', x.data_ptr(), kind, w.data_ptr(), b.data_ptr(), q[1:].data_ptr(),
                    scale[1:].data_ptr(), rows, windows, off.data_ptr(), channels, groups, 1e-5, EPI_SILU, ws.data_ptr(), need,
                    rt.stream())
        check_quantized(q[1:rows + 1], scale[1:rows + 1], x, w, b, groups, bounds, 'silu')
        assert (q[0] == 77).all() and (q[-1] == 77).all() and torch.isnan(scale[[0, rows + 1]]).all()


def test_conv_module_tail_keeps_other_rows(rt):
    """Rows of no window keep the residual stream they had, bit for bit, in place too."""
    rng = np.random.default_rng(3)
    for bounds in ([30, 40, 40, 155, 230], [100, 101], [0]):
        windows = len(bounds) - 1
        off = torch.tensor(bounds, dtype=torch.int32, device='cuda')
        x, w, b = inputs(4, 260, 1024, torch.float32)
        w8 = Int8Weight(dev(rng.integers(-127, 128, size=(1024, 1024)).astype(np.int8)), dev(rng.uniform(1e-3, 2e-3, 1024).astype(np.float32)))
        resid = dev(rng.normal(size=(260, 1024)).astype(np.float32))
        torch.full((64, 1 << 20), float('nan'), device='cuda')  # what a new tensor may find in its memory
        h = rt.group_norm_quantize(x, w, b, 32, windows=windows, offsets=off, epilogue=EPI_SILU)
        want = rt.linear_i8(h, w8, resid=resid, epilogue=EPI_RESIDUAL)
        for outside in (slice(0, bounds[0]), slice(bounds[-1], 260)):
            assert torch.equal(want[outside], resid[outside])
        stream = resid.clone()
        rt.linear_i8(h, w8, out=stream, resid=stream, epilogue=EPI_RESIDUAL)
        assert torch.equal(stream, want)
        assert not torch.equal(want[bounds[0]:bounds[-1]], resid[bounds[0]:bounds[-1]]) or bounds[0] == bounds[-1]


@pytest.mark.parametrize('rows,ragged', [(96, False), (96, True), (40, False), (3000, False)])
@pytest.mark.parametrize('channels', [4096, 16384])
def test_wide_groups_sum_by_column(rt, rows, channels, ragged):
    """One group of more columns than a CTA has threads for. Every column has one value in all rows, so its differences
    from its first row are 0, the sums are exact, and what is left are the roundings of the normalisation: x minus the mean,
    the scale and the multiply-add, one each, under 4 U |z| with the mean's remainder, U for that remainder's own. (Runs that mix these
    columns round the variance off by 28 U and the mean by 6 U deviations.)"""
    U = 2.0 ** -24
    value = np.array([-2.3483655, -0.90141344, -0.94846755, -1.0168121], np.float32)
    x = np.broadcast_to(np.resize(np.repeat(value, 1024), channels), (rows, channels))
    bounds = [3, rows - 5] if ragged else [0, rows]
    off = torch.tensor(bounds, dtype=torch.int32, device='cuda') if ragged else None
    w, b = torch.ones(channels, device='cuda'), torch.zeros(channels, device='cuda')
    got = f64(rt.group_norm(dev(x), w, b, 1, offsets=off))
    z = oi.group_norm(x, np.ones(channels), np.zeros(channels), 1, bounds)
    inside = slice(bounds[0], bounds[-1])
    assert (np.abs(got - z)[inside] <= U * (4 * np.abs(z) + 1)[inside]).all(), float(np.abs(got - z)[inside].max() / U)


def many_windows(ends):
    """Offsets of the windows that end at the rows ``ends``, each run of (row, how often)."""
    return torch.tensor(np.concatenate([[0]] + [np.full(n, r) for r, n in ends]).astype(np.int32), device='cuda')


@pytest.mark.parametrize('ends', [[(0, 300), (24, 1), (24, 300), (25, 1), (40, 700), (64, 2)],
                                  [(i, 1) for i in range(1, 65)], [(i, 257) for i in range(1, 65)],
                                  [(0, 1 << 21), (24, 1 << 21), (60, 1 << 20)]])
def test_many_windows(rt, ends):
    """Windows without rows between those with some, by the hundred and by the million. A million empty windows cost
    no more than a few: walked one after the other they took seconds, longer than the limit (4 s) of a wait in
    the product that follows. (The bound of 50 ms is a thousand times what the search takes.)"""
    off = many_windows(ends)
    rows, windows = 70, off.numel() - 1
    bounds = [0] + [r for r, _ in ends]
    for dtype, channels, groups, skip in ((torch.float32, 64, 4, 0), (torch.float16, 1040, 8, 0), (torch.float32, 64, 4, 1)):
        x, w, b = inputs(7, rows, channels, dtype, skip)
        out = torch.full_like(x, 9.0)
        rt.group_norm(x, w, b, groups, windows=windows, offsets=off, out=out)
        a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        rt.group_norm(x, w, b, groups, windows=windows, offsets=off, out=out)
        got = rt.group_norm_quantize(x, w, b, groups, windows=windows, offsets=off, epilogue=EPI_SILU)
        z.record()
        z.synchronize()
        assert a.elapsed_time(z) < 50.0
        want = oi.group_norm(f64(x), f64(w), f64(b), groups, bounds)[:bounds[-1]]
        fi = torch.finfo(dtype)
        # at most 64 rows: statistics and normalisation are off by under 64 x 2^-24 of the largest value
        bound = (fi.eps / 2 + 2.0 ** -18) * np.abs(want).max() + fi.tiny
        assert (np.abs(f64(out)[:bounds[-1]] - want) <= bound).all() and (out[bounds[-1]:] == 9).all()
        check_quantized(got.q, got.scale, x, w, b, groups, bounds, 'silu')


@pytest.mark.parametrize('windows,t,channels,groups,ragged,skip', [
    (1, 7, 1024, 32, False, 0), (8, 375, 1024, 32, False, 0), (3, 400, 1024, 1, False, 0), (5, 90, 1000, 8, False, 0), (2, 300, 35, 5, False, 0),
    (2, 3000, 64, 1, False, 0), (4, 200, 1000, 8, True, 0), (4, 200, 96, 96, True, 0), (3, 60, 8192, 2, False, 0), (2, 200, 64, 4, False, 1),
    (4, 2000, 256, 8, True, 1)])
def test_statistics_of_whole_numbers(rt, windows, t, channels, groups, ragged, skip):
    """Whole numbers from -8 to 24: every sum of differences and of their squares is a whole number below 2^24 and so
    exact in fp32, in whatever order, and the statistics are right to fp64. What is left is the normalisation: x minus the
    rounded mean, the scale and the multiply-add round once each, 3 U |z| (U = 2^-24), and what the mean's remainder
    loses is of the order of U^2; then half a step of the type. (32 differences of up to 32: sums below 2^10, squares below 2^15.)"""
    U = 2.0 ** -24
    rng = np.random.default_rng(channels + t)
    rows = windows * t
    bounds = sorted(rng.integers(0, rows + 1, windows + 1).tolist()) if ragged else [i * t for i in range(windows + 1)]
    off = torch.tensor(bounds, dtype=torch.int32, device='cuda') if ragged else None
    x = rng.integers(-8, 25, size=(rows, channels))
    z = oi.group_norm(x, np.ones(channels), np.zeros(channels), groups, bounds)[bounds[0]:bounds[-1]]
    w, b = torch.ones(channels, device='cuda'), torch.zeros(channels, device='cuda')
    for dtype in TYPES:
        flat = torch.zeros(rows * channels + skip, dtype=dtype, device='cuda')
        held = flat[skip:].view(rows, channels)
        held.copy_(dev(x.astype(np.float32)))
        got = f64(rt.group_norm(held, w, b, groups, windows=windows, offsets=off))[bounds[0]:bounds[-1]]
        err = 3.1 * U * np.abs(z) + 2.0 ** -40
        bound = err + (torch.finfo(dtype).eps / 2 * (np.abs(z) + err) if dtype != torch.float32 else 0.0)
        assert (np.abs(got - z) <= bound).all(), (dtype, float((np.abs(got - z) / bound).max()))
