"""SiLU and the GLU's gate over their whole range, in every kernel form of the 8-bit product and the group norm.

A masked channel has a bias of the type's lowest value, or minus infinity; its SiLU is 0 (NaN at minus infinity, the
product of an infinity and 0), and a gate there gives 0. Far below zero SiLU and sigmoid are z e^z and e^z.

Tolerance, U = 2^-24. The value z before the activation is off by at most dz (the product's 4 U (|acc s t| + |b|); the
group norm's bound of its own tests). It goes through the function itself, not through a common slope: SiLU falls
down to its minimum at -1.2785 and rises from there, so its values over [z - dz, z + dz] lie between those at the ends and, if inside,
the minimum; the sigmoid rises. The activation's own rounding: the exponent z log2(e) rounds twice (2 x 1.45 |z| U of
e^z after the factor ln 2 of 2^x: under 3 |z| U), and the exponential, the sum, the quotient and the product with z (or the
value) are under 8 U together. Numbers below 2^-126 may come out as 0: |z| 2^-126 (|a| 2^-126 for a gate), and nothing more past z = -128,
where e^z is far below 2^-126. Then half a step of the output's type.
"""
import numpy as np
import pytest
import torch

from oracle import int8 as oi
from parakeet_cuda_b200.pq8 import EPI_GLU, EPI_SILU
from parakeet_cuda_b200.runtime import Int8Weight, QuantizedRows, Runtime

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)
U = 2.0 ** -24
LOWEST = float(np.finfo(np.float32).min)
BIASES = np.array([0.0, -1.0, -8.0, -20.0, -43.0, -44.0, -50.0, -60.0, -80.0, -87.0, -88.0, -90.0, -100.0, -1e3, -1e5, -1e13,
                   -1e20, -1e30, LOWEST, -np.inf, 20.0, 50.0, 1e4, -46.0, -1e24, 3.0])
MIN_AT, MIN = -1.2784645427610738, -0.27846454276107374


@pytest.fixture(scope='module')
def rt():
    return Runtime(0)


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def f64(t):
    return t.double().cpu().numpy()


def silu(z):
    with np.errstate(invalid='ignore'):
        return z * oi.sigmoid(z)


def rounding(z):
    return (8 + 3 * np.minimum(np.maximum(-z, 0), 128)) * U


def silu_bound(z, dz):
    y = silu(z)
    err = np.maximum(np.abs(silu(z - dz) - y), np.abs(silu(z + dz) - y))
    err = np.where((z - dz < MIN_AT) & (z + dz > MIN_AT), np.maximum(err, y - MIN), err)
    return y, err + rounding(z) * (np.abs(y) + err) + np.minimum(np.abs(z), 128) * 2.0 ** -126


def gate_bound(a, da, g, dg):
    s = oi.sigmoid(g)
    ds = np.maximum(oi.sigmoid(g + dg) - s, s - oi.sigmoid(g - dg))
    err = np.abs(a) * ds + da * (s + ds)
    y = a * s
    return y, err + rounding(g) * (np.abs(y) + err) + (np.abs(a) + da) * 2.0 ** -126


def compare(got, y, bound):
    fi = torch.finfo(got.dtype)
    g = f64(got)
    nan = np.isnan(y)
    assert np.array_equal(np.isnan(g), nan), (np.argwhere(np.isnan(g) != nan)[:5], got.dtype)
    bound = bound + fi.eps / 2 * (np.abs(y) + bound) + fi.tiny * fi.eps
    bad = (np.abs(g - y) > bound) & ~nan
    assert not bad.any(), (int(bad.sum()), got.dtype, [(g[tuple(i)], y[tuple(i)], bound[tuple(i)]) for i in np.argwhere(bad)[:4]])


# the GEMV, single-CTA tiles, split K and CTA pairs
@pytest.mark.parametrize('m,k', [(1, 64), (8, 64), (9, 64), (50, 2064), (200, 64), (3000, 144)])
@pytest.mark.parametrize('dtype', TYPES)
def test_product(rt, m, k, dtype):
    rng = np.random.default_rng(m)
    n = 1024 if m > 1000 else 2 * len(BIASES)
    w = rng.integers(-127, 128, size=(n, k)).astype(np.int8)
    q = rng.integers(-127, 128, size=(m, k)).astype(np.int8)
    s, t = rng.uniform(.5, 1, m).astype(np.float32), (rng.uniform(.5, 1, n) / (5000 * k ** .5)).astype(np.float32)
    bias = np.resize(BIASES, n).astype(np.float32)
    x8, w8 = QuantizedRows(dev(q), dev(s)), Int8Weight(dev(w), dev(t))
    z, size = oi.product(q, s, w, t, bias)
    dz = np.where(np.isfinite(size), 4 * U * size, 0.0)
    compare(rt.linear_i8(x8, w8, bias=dev(bias), epilogue=EPI_SILU, out_dtype=dtype), *silu_bound(z, dz))
    half = n // 2
    bias[:half], bias[half:] = rng.normal(size=half), np.resize(BIASES, half)
    z, size = oi.product(q, s, w, t, bias)
    dz = np.where(np.isfinite(size), 4 * U * size, 0.0)
    got = rt.linear_i8(x8, w8, bias=dev(bias), epilogue=EPI_GLU, out_dtype=dtype)
    compare(got, *gate_bound(z[:, :half], dz[:, :half], z[:, half:], dz[:, half:]))
    assert rt.device_status() == 0


# one launch; units that straddle groups; single columns; two launches (ragged); a misaligned x
@pytest.mark.parametrize('channels,groups,windows,skip,ragged', [(64, 4, 3, 0, False), (104, 8, 2, 0, False), (35, 5, 2, 0, False),
                                                                 (64, 4, 4, 0, True), (64, 4, 3, 1, False)])
@pytest.mark.parametrize('dtype', TYPES)
def test_group_norm(rt, channels, groups, windows, skip, ragged, dtype):
    rng = np.random.default_rng(channels + windows)
    rows = 20 * windows
    flat = dev(rng.normal(size=rows * channels + skip).astype(np.float32), dtype)
    x = flat[skip:].view(rows, channels)
    w, b = (1 + 0.2 * rng.normal(size=channels)).astype(np.float32), np.resize(BIASES, channels).astype(np.float32)
    bounds = [0, 7, 30, 31, rows] if ragged else [20 * i for i in range(windows + 1)]
    off = torch.tensor(bounds, dtype=torch.int32, device='cuda') if ragged else None
    got = rt.group_norm(x, dev(w), dev(b), groups, windows=windows, offsets=off, epilogue=EPI_SILU)
    plain = oi.group_norm(f64(x), np.ones(channels), np.zeros(channels), groups, bounds)
    far = 2 * np.abs(plain).max()  # D of the group norm's tolerance, in deviations
    wz = np.abs(plain * w)
    with np.errstate(invalid='ignore', over='ignore'):
        dz = U * (6 * (2 * wz + 2 * np.abs(b)) + 18 * far * np.abs(w) + 28 * far ** 2 * wz)
    z = plain * w + b
    compare(got, *silu_bound(z, np.where(np.isfinite(dz), dz, 0.0)))


@pytest.mark.parametrize('windows,ragged', [(3, False), (4, True)])
@pytest.mark.parametrize('channels,groups', [(64, 4), (1024, 32)])
def test_group_norm_quantize(rt, windows, ragged, channels, groups):
    """Masked channels are 0 and do not touch their rows' scale, in the form of one launch and of two."""
    rng = np.random.default_rng(channels + windows)
    rows = 20 * windows
    x = dev(rng.normal(size=(rows, channels)).astype(np.float32))
    w, b = (1 + 0.2 * rng.normal(size=channels)).astype(np.float32), np.zeros(channels, np.float32)
    masked = [-60.0, -1e5, -1e13, -1e20, -1e30, LOWEST]
    bounds = [0, 7, 30, 31, rows] if ragged else [20 * i for i in range(windows + 1)]
    off = torch.tensor(bounds, dtype=torch.int32, device='cuda') if ragged else None
    x[:, 3::8] -= 4  # always below the mean
    for value in masked + [1e20, 1e22]:  # a bias, or a weight that takes the value there
        b[3::8], w[3::8] = (value, 1.0) if value < 0 else (0.0, value)
        got = rt.group_norm_quantize(x, dev(w), dev(b), groups, windows=windows, offsets=off, epilogue=EPI_SILU)
        q, s, margin = oi.quantize(oi.group_norm(f64(x), w, b, groups, bounds, epilogue='silu'))
        np.testing.assert_allclose(got.scale.cpu().numpy(), s, rtol=2.0 ** -23, atol=0)
        wrong = got.q.cpu().numpy() != q
        assert not (wrong & (margin > 1e-9)).any(), (value, int(wrong.sum()))
