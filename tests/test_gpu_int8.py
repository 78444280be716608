"""GPU parity of the row quantisation and the 8-bit product against the 64-bit oracle.

Tolerances. The integers of a quantised row are exact: equal to the oracle's, except that with a
norm in front a value whose quotient lies within 1e-9 of a border may fall either way (both
sides compute in fp64, whose roundings here are below 1e-12 of the quotient's scale). Products:
the integer sum is exact; its conversion to fp32, the multiplication by the token's scale and the
multiply-add with the channel's scale and bias round once each, so |err| <= 4 x 2^-24 x (|acc s t|
+ |b|) before the activation. SiLU and the GLU's gate add their own rounding (expf, one sum, one
quotient: under 8 x 2^-24 of the result) and pass the error of z on with a slope of at most 1.1; the output's
rounding is half a step of its type.
"""
import ctypes as C
import subprocess
import sys
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import int8 as oi
from oracle import q8
from parakeet_cuda_b200 import pq8
from parakeet_cuda_b200.pq8 import EPI_GLU, EPI_NONE, EPI_RELU, EPI_RESIDUAL, EPI_SILU
from parakeet_cuda_b200.runtime import Int8Weight, QuantizedRows, Runtime
from parakeet_cuda_b200.synthetic import q8_0_blocks

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)
U = 2.0 ** -24


@pytest.fixture(scope='module')
def rt():
    return Runtime(0)


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda().to(dtype) if dtype else \
        torch.from_numpy(np.ascontiguousarray(a)).cuda()


def f64(t):
    return t.double().cpu().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tokens(rng, rows, width, dtype):
    x = rng.normal(size=(rows, width)) * np.exp(rng.normal(size=(rows, 1))) + 0.3 * rng.normal(size=(1, width))
    return dev(x.astype(np.float32), dtype)


def check_rows(got, h, borders):
    q, s, margin = oi.quantize(h)
    np.testing.assert_array_equal(got.scale.cpu().numpy(), s)
    gq = got.q.cpu().numpy()
    wrong = gq != q
    assert not (wrong & (margin > borders)).any(), (int(wrong.sum()), float(margin[wrong].max()))
    assert (np.abs(gq.astype(int) - q.astype(int)) <= 1).all()


# the three forms of the row kernel (a warp, a CTA, a CTA reading again) and their edges
WIDTHS = (16, 48, 640, 1024, 1040, 4096, 8192, 8208, 20000)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width', WIDTHS)
@pytest.mark.parametrize('norm', [False, True])
def test_quantize_rows(rt, width, dtype, norm):
    rng = np.random.default_rng(width + norm)
    rows = 37 if width <= 1024 else 5
    x = tokens(rng, rows, width, dtype)
    w, b = dev((1 + 0.2 * rng.normal(size=width)).astype(np.float32)), dev(0.2 * rng.normal(size=width).astype(np.float32))
    got = rt.quantize_rows(x, norm=(w, b) if norm else None)
    h = oi.layer_norm(f64(x), f64(w), f64(b)) if norm else f64(x)
    check_rows(got, h, 1e-9 if norm else -1.0)


@pytest.mark.parametrize('width', [1024, 4096, 16384])
def test_quantize_rows_borders(rt, width):
    """Values on and next to the border between two integers, against rational arithmetic."""
    rng = np.random.default_rng(width)
    rows = 4
    x = np.zeros((rows, width), np.float32)
    for r in range(rows):
        top = np.float32(127.0 if r == 0 else rng.uniform(0.5, 300.0))
        s = np.float32(top / np.float32(127.0))
        mid = (rng.integers(-126, 126, width) + 0.5).astype(np.float64) * np.float64(s)
        v = mid.astype(np.float32)
        step = rng.integers(-1, 2, width)
        v = np.where(step < 0, np.nextafter(v, np.float32(-np.inf)), np.where(step > 0, np.nextafter(v, np.float32(np.inf)), v))
        v[0] = top
        x[r] = v
    got = rt.quantize_rows(dev(x))
    q = got.q.cpu().numpy()
    for r in range(rows):
        s = Fraction(float(np.float32(np.abs(x[r]).max() / np.float32(127.0))))
        want = [round(Fraction(float(v)) / s) for v in x[r]]  # ties to even
        np.testing.assert_array_equal(q[r], np.clip(want, -127, 127))


@pytest.mark.parametrize('width', [64, 2048, 8208])
@pytest.mark.parametrize('norm', [False, True])
def test_quantize_rows_odd_values(rt, width, norm):
    """Zero rows, constant rows, single values, infinities, NaN, rows near both ends of fp32's range."""
    rng = np.random.default_rng(3)
    x = rng.normal(size=(11, width)).astype(np.float32)
    x[0] = 0
    x[1] = 0
    x[1, width // 2] = -3.0
    x[2, 5] = np.inf
    x[3, 7] = -np.inf
    x[4, 9] = np.nan
    x[5] *= 1e-41  # subnormal: the scale has a few bits, or none
    x[6] *= 1e-37
    x[7] *= 1e-30
    x[8] *= 1e37 / 8
    x[9] = 1e6 + x[9]
    w, b = np.ones(width, np.float32), np.zeros(width, np.float32)
    got = rt.quantize_rows(dev(x), norm=(dev(w), dev(b)) if norm else None)
    with np.errstate(all='ignore'):
        h = oi.layer_norm(x, w, b) if norm else x.astype(np.float64)
        h[2:5] = np.nan
        check_rows(got, h, 1e-9 if norm else -1.0)
    again = rt.quantize_rows(dev(x), norm=(dev(w), dev(b)) if norm else None)
    assert torch.equal(got.q, again.q)


def test_quantize_rows_strides_and_sizes(rt):
    """A slice of wider rows, rows that start off a 16-byte boundary, one row, none, the widest."""
    rng = np.random.default_rng(4)
    big = dev(rng.normal(size=(9, 333)).astype(np.float32))
    for dtype in TYPES:
        x = big.to(dtype)
        for view in (x[:, 3:67], x[:, :64], x[1:2, 5:101], x[:0, :64], x[::2, 16:48]):
            got = rt.quantize_rows(view)
            assert got.q.shape == view.shape
            if view.shape[0]:
                check_rows(got, f64(view), -1.0)
    wide = dev(rng.normal(size=(2, pq8.I8_MAX_K)).astype(np.float32))
    check_rows(rt.quantize_rows(wide), f64(wide), -1.0)


def weights(rng, n, k, full=False):
    q = rng.integers(-128 if full else -127, 128, size=(n, k)).astype(np.int8)
    return q, (rng.uniform(0.5, 2.0, n) * 1e-3).astype(np.float32)


EPIS = {'none': EPI_NONE, 'relu': EPI_RELU, 'silu': EPI_SILU, 'glu': EPI_GLU, 'residual': EPI_RESIDUAL}


def expected(z, size, epi, resid, alpha, dtype):
    """(value, bound) of an output whose z is off by at most 4 x 2^-24 x size."""
    dz = 4 * U * size
    if epi == 'glu':
        h = z.shape[1] // 2
        s = oi.sigmoid(z[:, h:])
        y = z[:, :h] * s
        err = dz[:, :h] * s + np.abs(z[:, :h]) * 0.25 * dz[:, h:] + 8 * U * np.abs(y) + 1.1 * dz[:, :h] * dz[:, h:]
    elif epi == 'silu':
        y = z * oi.sigmoid(z)
        err = 1.1 * dz + 8 * U * np.abs(y)
    elif epi == 'residual':
        y = resid + alpha * z
        err = abs(alpha) * dz + U * np.abs(y)
    else:
        y, err = oi.act(z, epi), dz
    tiny = float(torch.finfo(dtype).tiny) * torch.finfo(dtype).eps  # a step of the subnormals
    return y, err + half_step(dtype) * (np.abs(y) + err) + tiny + 1e-37


def check_product(got, q, s, w, t, bias, epi, resid, alpha):
    z, size = oi.product(q, s, w, t, bias)
    y, bound = expected(z, size, epi, resid, alpha, got.dtype)
    g = f64(got)
    nan = np.isnan(y)
    assert np.array_equal(np.isnan(g), nan)
    bad = np.abs(g - y)[~nan] > bound[~nan]
    assert not bad.any(), (int(bad.sum()), float((np.abs(g - y)[~nan] / bound[~nan]).max()))


# below, at and above the row counts at which another kernel or tile takes over; odd channels; K
# that ends inside a 128-byte block, one block and many
SHAPES = [(1, 16, 1), (1, 1024, 4096), (2, 48, 130), (3, 640, 8198), (5, 4096, 1024), (8, 640, 33), (9, 144, 257),
          (16, 1024, 1024), (17, 112, 129), (33, 2064, 300), (64, 4096, 640), (65, 1024, 2048), (128, 256, 4096),
          (129, 640, 65), (257, 176, 514), (375, 1024, 2048), (700, 128, 700), (1300, 1040, 1026)]


@pytest.mark.parametrize('m,k,n', SHAPES)
@pytest.mark.parametrize('epi', list(EPIS))
def test_gemm_i8(rt, m, k, n, epi):
    rng = np.random.default_rng(m * 7 + k + n)
    if epi == 'glu':
        n += n % 2
    out = n // 2 if epi == 'glu' else n
    w, t = weights(rng, n, k, full=True)
    q = rng.integers(-128, 128, size=(m, k)).astype(np.int8)
    s = rng.uniform(0.5, 2.0, m).astype(np.float32) * np.float32(1e-2)
    dtype = TYPES[(m + k + len(epi)) % 3]
    bias = None if m % 2 else rng.normal(size=n).astype(np.float32)
    resid = dev(rng.normal(size=(m, out)).astype(np.float32), dtype) if epi == 'residual' else None
    y = rt.linear_i8(QuantizedRows(dev(q), dev(s)), Int8Weight(dev(w), dev(t)),
                     bias=None if bias is None else dev(bias), resid=resid, epilogue=EPIS[epi], alpha=0.5,
                     out_dtype=dtype)
    check_product(y, q, s, w, t, bias, epi, None if resid is None else f64(resid), 0.5)
    assert rt.device_status() == 0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m', [1, 6, 40, 300])
def test_gemm_i8_extreme_sums(rt, dtype, m):
    """The largest sums that 32 bits hold, of both signs, and the widest K."""
    k, n = pq8.I8_MAX_K, 3
    w = np.full((n, k), -128, np.int8)
    w[1] = 127
    q = np.full((m, k), -128, np.int8)
    q[m // 2:] = 127
    s, t = np.full(m, 2.0 ** -20, np.float32), np.full(n, 2.0 ** -6, np.float32)
    y = rt.linear_i8(QuantizedRows(dev(q), dev(s)), Int8Weight(dev(w), dev(t)), out_dtype=dtype)
    check_product(y, q, s, w, t, None, 'none', None, 1.0)


@pytest.mark.parametrize('x_type', TYPES)
@pytest.mark.parametrize('norm', [False, True])
@pytest.mark.parametrize('m,k,n', [(1, 640, 2560), (7, 1024, 1024), (8, 4096, 640), (12, 64, 48), (200, 1024, 512),
                                   (5, 9008, 32)])
def test_linear_i8(rt, m, k, n, norm, x_type):
    """Float tokens to float outputs: the integers the oracle finds for the tokens, then the product's
    bound (no value of these inputs lies within 1e-9 of a border: checked)."""
    rng = np.random.default_rng(m + k + n)
    x = tokens(rng, m, k, x_type)
    w, t = weights(rng, n, k)
    g, b = (1 + 0.1 * rng.normal(size=k)).astype(np.float32), (0.1 * rng.normal(size=k)).astype(np.float32)
    h = oi.layer_norm(f64(x), g, b) if norm else f64(x)
    q, s, margin = oi.quantize(h)
    if norm:
        assert margin.min() > 1e-9
    bias = rng.normal(size=n).astype(np.float32)
    y = rt.linear_i8(x, Int8Weight(dev(w), dev(t)), bias=dev(bias), epilogue=EPI_SILU,
                     norm=(dev(g), dev(b)) if norm else None)
    check_product(y, q, s, w, t, bias, 'silu', None, 1.0)


def test_linear_i8_bad_rows_stay_alone(rt):
    """A token row with an infinity or a NaN gives NaN outputs; its neighbours are what they are without it."""
    rng = np.random.default_rng(8)
    for m in (4, 50, 300):
        x = rng.normal(size=(m, 256)).astype(np.float32)
        w, t = weights(rng, 200, 256)
        w8 = Int8Weight(dev(w), dev(t))
        clean = rt.linear_i8(dev(x), w8)
        x[1, 3], x[m - 1, 200] = np.nan, np.inf
        got = rt.linear_i8(dev(x), w8)
        assert torch.isnan(got[1]).all() and torch.isnan(got[m - 1]).all()
        keep = [i for i in range(m) if i not in (1, m - 1)]
        assert torch.equal(got[keep], clean[keep])


def test_gemm_i8_writes_only_its_output(rt):
    """Rows and columns around the output keep their bytes; the residual may be the output."""
    rng = np.random.default_rng(9)
    for m, n in ((1, 100), (8, 33), (9, 130), (70, 257), (300, 65)):
        k = 320
        w, t = weights(rng, n, k)
        q = rng.integers(-127, 128, size=(m, k)).astype(np.int8)
        s = rng.uniform(0.5, 1, m).astype(np.float32)
        for dtype in TYPES:
            buf = torch.full((m + 2, n), 7.0, dtype=dtype, device='cuda')
            rt.linear_i8(QuantizedRows(dev(q), dev(s)), Int8Weight(dev(w), dev(t)), out=buf[1:m + 1])
            assert (buf[0] == 7).all() and (buf[m + 1] == 7).all()
            check_product(buf[1:m + 1], q, s, w, t, None, 'none', None, 1.0)
        r = dev(rng.normal(size=(m, n)).astype(np.float32))
        old = f64(r)
        rt.linear_i8(QuantizedRows(dev(q), dev(s)), Int8Weight(dev(w), dev(t)), out=r, resid=r, epilogue=EPI_RESIDUAL,
                     alpha=-2.0)
        check_product(r, q, s, w, t, None, 'residual', old, -2.0)


def test_int8_weight_from_q8_0(rt):
    rng = np.random.default_rng(10)
    n, k = 130, 96
    raw = q8_0_blocks(rng, n, k)
    w8 = rt.int8_weight((raw, n, k))
    check_rows(QuantizedRows(w8.q, w8.scale), q8.decode(raw, n, k).astype(np.float64), -1.0)
    same = rt.int8_weight(dev(q8.decode(raw, n, k).astype(np.float32)))
    assert torch.equal(same.q, w8.q) and torch.equal(same.scale, w8.scale)


def test_linear_i8_graph_streams_and_order(rt):
    """One captured graph of two calls, replayed on new inputs, and calls on two streams at once, give the
    eager results bit for bit; the weights may be quantised right before their use."""
    rng = np.random.default_rng(11)
    for m in (1, 8, 40, 500):
        w1 = dev(rng.normal(size=(512, 256)).astype(np.float32))
        w2 = dev(rng.normal(size=(256, 512)).astype(np.float32))
        x = dev(rng.normal(size=(m, 256)).astype(np.float32))

        def step():
            a, b = rt.int8_weight(w1), rt.int8_weight(w2)
            hidden = rt.linear_i8(x, a, epilogue=EPI_SILU, out_dtype=torch.bfloat16)
            return rt.linear_i8(hidden, b, resid=x, epilogue=EPI_RESIDUAL)

        eager = step().clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
        x.copy_(dev(rng.normal(size=(m, 256)).astype(np.float32)))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = [[], []]
        torch.cuda.synchronize()
        for _ in range(5):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    outs[i].append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for side in outs for o in side)
    assert rt.device_status() == 0


def test_linear_i8_refuses(rt):
    x = torch.zeros(4, 64, device='cuda')
    w8 = Int8Weight(torch.zeros(32, 64, dtype=torch.int8, device='cuda'), torch.ones(32, device='cuda'))
    g = torch.ones(64, device='cuda')
    ok = rt.linear_i8(x, w8)
    assert not ok.any()
    bad = [lambda: rt.linear_i8(x.double(), w8), lambda: rt.linear_i8(x.cpu(), w8), lambda: rt.linear_i8(x[0], w8),
           lambda: rt.linear_i8(x.t(), w8), lambda: rt.linear_i8(x[:, :48], w8), lambda: rt.linear_i8(x[:1].expand(4, 64), w8),
           lambda: rt.linear_i8(x, Int8Weight(w8.q.float(), w8.scale)),
           lambda: rt.linear_i8(x, Int8Weight(w8.q, w8.scale[:31])),
           lambda: rt.linear_i8(x, w8, bias=torch.zeros(31, device='cuda')),
           lambda: rt.linear_i8(x, w8, bias=torch.zeros(32, device='cuda', dtype=torch.float16)),
           lambda: rt.linear_i8(x, w8, out=torch.zeros(4, 31, device='cuda')),
           lambda: rt.linear_i8(x, w8, out=torch.zeros(4, 64, device='cuda')[:, ::2]),
           lambda: rt.linear_i8(x, w8, out=torch.zeros(4, 32, device='cuda'), out_dtype=torch.float16),
           lambda: rt.linear_i8(x, w8, out_dtype=torch.float64),
           lambda: rt.linear_i8(x, w8, epilogue=EPI_RESIDUAL, resid=torch.zeros(4, 32, device='cuda', dtype=torch.float16)),
           lambda: rt.linear_i8(x, w8, norm=(g, g.double())), lambda: rt.linear_i8(x, w8, norm=(g[:32], g[:32])),
           lambda: rt.linear_i8(rt.quantize_rows(x), w8, norm=(g, g)), lambda: rt.quantize_rows(x.int())]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    for f in (lambda: rt.linear_i8(x, w8, epilogue=EPI_RESIDUAL), lambda: rt.linear_i8(x, w8, epilogue=9),
              lambda: rt.quantize_rows(torch.zeros(2, 24, device='cuda'))):
        with pytest.raises(pq8.PQ8Error):
            f()
    assert rt.linear_i8(x[:0], w8).shape == (0, 32)
    assert rt.linear_i8(rt.quantize_rows(x[:0]), w8).shape == (0, 32)


def test_linear_i8_nan_passes_every_epilogue(rt):
    """A bad row, a bad channel and a bad gate reach the output through every activation, and nothing else."""
    rng = np.random.default_rng(12)
    n, k = 192, 256
    w, t = weights(rng, n, k)
    bad_t = t.copy()
    bad_t[100] = np.nan  # for the GLU: the gate of channel 4
    for m in (3, 20, 300):
        x = rng.normal(size=(m, k)).astype(np.float32)
        x[1, 7] = np.inf
        for epi in (EPI_NONE, EPI_RELU, EPI_SILU, EPI_GLU):
            clean = rt.linear_i8(dev(np.delete(x, 1, 0)), Int8Weight(dev(w), dev(t)), epilogue=epi)
            got = rt.linear_i8(dev(x), Int8Weight(dev(w), dev(bad_t)), epilogue=epi)
            assert torch.isnan(got[1]).all()
            col = 4 if epi == EPI_GLU else 100
            assert torch.isnan(got[:, col]).all()
            rest = torch.cat([got[:1], got[2:]])
            keep = [j for j in range(got.shape[1]) if j != col]
            if epi in (EPI_NONE, EPI_RELU):
                assert torch.equal(rest[:, keep], clean[:, keep])
            else:
                # two tokens' sigmoids share one reciprocal, and without the bad row other tokens are
                # neighbours: each side is within 8 U |y| of the same z's activation (module docstring)
                a, b = f64(rest[:, keep]), f64(clean[:, keep])
                assert (np.abs(a - b) <= 8 * U * (np.abs(a) + np.abs(b)) + 2.0 ** -62).all()


def test_int8_weight_whose_memory_changes(rt):
    """A weight can be written in place or given other memory of its size; memory of another is refused."""
    q, s = torch.ones(32, 64, dtype=torch.int8, device='cuda'), torch.ones(32, device='cuda')
    w8 = Int8Weight(q, s)
    x = torch.ones(9, 64, device='cuda')
    a = rt.linear_i8(x, w8)
    w8.q.fill_(2)
    assert torch.equal(rt.linear_i8(x, w8), 2 * a)
    q.data = torch.full((32, 64), 3, dtype=torch.int8, device='cuda')
    assert torch.equal(rt.linear_i8(x, w8), 3 * a)
    for bad in (torch.ones(16, 64, dtype=torch.int8, device='cuda'), torch.ones(1, 64, dtype=torch.int8, device='cuda').expand(32, 64)):
        q.data = bad
        with pytest.raises(ValueError):
            rt.linear_i8(x, w8)
    q.data = torch.ones(32, 64, dtype=torch.int8, device='cuda')
    s.data = torch.ones(31, device='cuda')
    with pytest.raises(ValueError):
        rt.linear_i8(x, w8)


FIRST_CALL = """
import torch
from parakeet_cuda_b200.runtime import Int8Weight, Runtime
rt = Runtime(0)
torch.manual_seed(0)
w8 = Int8Weight(torch.randint(-127, 128, (512, 4096), dtype=torch.int8, device='cuda'), torch.rand(512, device='cuda'))
gw, gb = torch.rand(4096, device='cuda'), torch.rand(4096, device='cuda')
xs = [torch.randn(m, 4096, device='cuda') for m in (1, 5, 60, 400, 2500)]
def step():
    out = [rt.linear_i8(x, w8, norm=(gw, gb)) for x in xs]
    for x in xs:
        out.append(rt.group_norm(x, gw, gb, 32))
        out.append(rt.group_norm_quantize(x, gw, gb, 32).scale)
    return out
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
assert rt.device_status() == 0
print('same')
"""


def test_first_calls_captured():
    """A process whose first calls are captured: per-device state is made under capture, same bits as eager."""
    root = Path(__file__).resolve().parent.parent
    run = subprocess.run([sys.executable, '-c', FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and 'same' in run.stdout, run.stderr[-2000:]


def test_two_graphs_in_flight(rt):
    """Two captured graphs replayed on two streams at once, each with its own scratch."""
    rng = np.random.default_rng(13)
    w8 = rt.int8_weight(dev(rng.normal(size=(1024, 1024)).astype(np.float32)))
    g, b = dev(rng.normal(size=1024).astype(np.float32)), dev(rng.normal(size=1024).astype(np.float32))
    xs = [dev(rng.normal(size=(700, 1024)).astype(np.float32)) for _ in range(2)]
    made = []
    for x in xs:
        want = rt.linear_i8(rt.group_norm_quantize(x, g, b, 4), w8, resid=x, epilogue=EPI_RESIDUAL)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = x
            for _ in range(4):
                y = rt.linear_i8(rt.group_norm_quantize(x, g, b, 4), w8, resid=x, epilogue=EPI_RESIDUAL)
        made.append((graph, y, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, _, _, st in made:
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, y, want, _ in made:
        assert torch.equal(y, want)


def test_past_32_bit_offsets(rt):
    """Tokens, integers and outputs of more than 2^31 elements: the last rows are what they are alone."""
    rng = np.random.default_rng(14)
    torch.manual_seed(14)
    w, t = weights(rng, 8192, 64)
    w8 = Int8Weight(dev(w), dev(t))
    m = (1 << 31) // 8192 + 500
    x = torch.randn(m, 64, device='cuda')
    y = rt.linear_i8(x, w8, out_dtype=torch.bfloat16)
    for part in (slice(0, 300), slice(m - 300, m)):
        assert torch.equal(y[part], rt.linear_i8(x[part], w8, out_dtype=torch.bfloat16))
    del y
    m = (1 << 31) // 4096 + 70
    x = torch.randn(m, 4096, device='cuda', dtype=torch.float16)
    got = rt.quantize_rows(x)
    alone = rt.quantize_rows(x[m - 90:])
    assert torch.equal(got.q[m - 90:], alone.q) and torch.equal(got.scale[m - 90:], alone.scale)
    w, t = weights(rng, 48, 4096)
    w8 = Int8Weight(dev(w), dev(t))
    y, z = rt.linear_i8(got, w8), rt.linear_i8(alone, w8)
    assert torch.equal(y[m - 90:], z)
    far = torch.empty_strided((9, 64), (1 << 29, 1), dtype=torch.float16, device='cuda')  # rows 1 GB apart
    far.copy_(x[:9, :64])
    near = rt.quantize_rows(x[:9, :64].contiguous())
    got = rt.quantize_rows(far)
    assert torch.equal(got.q, near.q) and torch.equal(got.scale, near.scale)


def test_int8_rows_whose_memory_leaves_the_device(rt):
    """Weights and tokens whose tensors were moved to the host after they were made are refused, not read."""
    x = torch.ones(9, 64, device='cuda')
    for part in ('q', 'scale'):
        w8 = Int8Weight(torch.ones(32, 64, dtype=torch.int8, device='cuda'), torch.ones(32, device='cuda'))
        rows = rt.quantize_rows(x)
        want = rt.linear_i8(rows, w8)
        for held in (w8, rows):
            t = getattr(held, part)
            kept = t.data
            t.data = t.cpu()
            with pytest.raises(ValueError):
                rt.linear_i8(rows, w8)
            t.data = kept
        assert torch.equal(rt.linear_i8(rows, w8), want)
    with pytest.raises(ValueError):
        rt.linear_i8(x.cpu(), w8)


def test_int8_weight_refuses_partial_blocks(rt):
    """Q8_0 rows that are not whole blocks: two rows of 16 are no block of 32."""
    blocks = q8_0_blocks(np.random.default_rng(1), 3, 32)
    assert rt.int8_weight((blocks, 3, 32)).k == 32
    for count, n, k in ((2, 4, 16), (3, 2, 48), (1, 2, 16), (2, 3, 32)):  # (the last: too few bytes)
        with pytest.raises(ValueError):
            rt.int8_weight((blocks[:count], n, k))
