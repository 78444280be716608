"""Every tile of the 8-bit product against the integer oracle: single CTAs of 16 to 128 tokens with K in one piece
and in 2, 4 and 8, and pairs of 192 and 256, in one wave and in several. Each case says which tile it is for, so that a
change of the tile model cannot leave one untested.

The sums are exact in float64 (below 2^31) and are taken on the GPU by torch. Tolerance, U = 2^-24: as in test_gpu_int8.py, dz = 4 U (|acc s t| +
|b|) before the activation, a slope of at most 1.1, 8 U of the result for SiLU and gates, U for the residual's sum, half a step of the type.
"""
import pytest
import torch

from parakeet_cuda_b200.pq8 import EPI_GLU, EPI_NONE, EPI_RELU, EPI_RESIDUAL, EPI_SILU
from parakeet_cuda_b200.runtime import Int8Weight, QuantizedRows, Runtime

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)
EPIS = {'none': EPI_NONE, 'relu': EPI_RELU, 'silu': EPI_SILU, 'glu': EPI_GLU, 'residual': EPI_RESIDUAL}
U = 2.0 ** -24


@pytest.fixture(scope='module')
def rt():
    return Runtime(0)


# tile (tokens, CTAs, K splits): m, n, k. Pairs: ragged m; odd numbers of 128-channel tiles (a pair's second CTA has none)
# and even ones; channels that end inside a tile; K that ends inside a block of 128; one, two and three tiles per pair. For the GLU, halves
# of a multiple of 16 (one load of values and gates) and others.
CASES = [
    ((16, 1, 1), 9, 34, 112), ((16, 1, 2), 9, 8198, 2064), ((16, 1, 4), 9, 34, 2064), ((16, 1, 8), 13, 34, 4096),
    ((32, 1, 1), 65, 4096, 112), ((32, 1, 2), 23, 8198, 2064), ((32, 1, 4), 700, 34, 2064), ((32, 1, 8), 289, 34, 4096),
    ((64, 1, 1), 198, 8198, 112), ((64, 1, 2), 37, 8198, 4096), ((64, 1, 4), 700, 130, 2064), ((64, 1, 8), 700, 34, 4096),
    ((128, 1, 1), 135, 8198, 640), ((128, 1, 2), 65, 8198, 4096), ((128, 1, 4), 65, 4096, 4096), ((128, 1, 8), 700, 130, 9008),
    ((192, 2, 1), 2500, 1026, 1040), ((192, 2, 1), 2999, 1024, 1024), ((192, 2, 1), 1499, 4094, 208), ((192, 2, 1), 4500, 2050, 176),
    ((192, 2, 1), 1499, 4096, 208),
    ((256, 2, 1), 3500, 1026, 1040), ((256, 2, 1), 1499, 8198, 640), ((256, 2, 1), 2999, 4094, 208), ((256, 2, 1), 2999, 4096, 208),
    ((256, 2, 1), 2000, 2050, 176),
]


def expected(acc, s, t, bias, epi, resid, alpha):
    """(value, bound) in float64."""
    p = acc * s.double()[:, None] * t.double()
    z, dz = p + bias.double(), 4 * U * (p.abs() + bias.double().abs())
    if epi == 'glu':
        half = z.shape[1] // 2
        a, sig, da, dg = z[:, :half], torch.sigmoid(z[:, half:]), dz[:, :half], dz[:, half:]
        y = a * sig
        return y, da * sig + a.abs() * 0.25 * dg + 1.1 * da * dg + 8 * U * y.abs()
    if epi == 'silu':
        y = z * torch.sigmoid(z)
        return y, 1.1 * dz + 8 * U * y.abs()
    if epi == 'residual':
        y = resid.double() + alpha * z
        return y, abs(alpha) * dz + U * y.abs()
    return (z.clamp(min=0) if epi == 'relu' else z), dz


@pytest.mark.parametrize('tile,m,n,k', CASES)
@pytest.mark.parametrize('epi', list(EPIS))
def test_tile(rt, tile, m, n, k, epi):
    assert rt.lib.gemm_i8_tile(m, n, k, EPIS[epi]) == tile
    g = torch.Generator(device='cuda').manual_seed(m + n + k)
    ints = lambda *shape: torch.randint(-128, 128, shape, generator=g, device='cuda', dtype=torch.int8)
    uniform = lambda *shape: 0.5 + 1.5 * torch.rand(*shape, generator=g, device='cuda')
    q, w = ints(m, k), ints(n, k)
    s, t = 1e-2 * uniform(m), uniform(n) / (50 * k ** 0.5)
    dtype = TYPES[(m + n + len(epi)) % 3]
    out = n // 2 if epi == 'glu' else n
    bias = torch.randn(n, generator=g, device='cuda')
    resid = torch.randn(m, out, generator=g, device='cuda').to(dtype) if epi == 'residual' else None
    buf = torch.full((m + 2, out), 7.0, dtype=dtype, device='cuda')
    rt.linear_i8(QuantizedRows(q, s), Int8Weight(w, t), out=buf[1:m + 1], bias=bias, resid=resid, epilogue=EPIS[epi], alpha=0.5)
    y, err = expected(q.double() @ w.double().T, s, t, bias, epi, resid, 0.5)
    fi = torch.finfo(dtype)
    bound = err + fi.eps / 2 * (y.abs() + err) + fi.tiny * fi.eps + 1e-37
    bad = (buf[1:m + 1].double() - y).abs() > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), bad.nonzero()[-4:].tolist())
    assert (buf[0] == 7).all() and (buf[m + 1] == 7).all()  # rows around the output keep their bytes
    assert rt.device_status() == 0


def test_few_tokens_take_no_tile(rt):
    assert rt.lib.gemm_i8_tile(8, 4096, 1024) == (0, 1, 1)
    assert rt.lib.gemm_i8_tile(9, 4096, 1024)[0] > 0
