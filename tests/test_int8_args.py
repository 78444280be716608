"""Refusals of the 8-bit product and group norm entry points that need no GPU: shapes, types,
alignment, overlaps and workspaces are checked before a device is touched. (Addresses below are
made up and never read.)"""
import ctypes as C

import numpy as np
import pytest

from oracle import int8 as oi
from parakeet_cuda_b200 import pq8

X, W, Q, S, Y, B, WS = (0x10000000 * (i + 1) for i in range(7))
BIG = 1 << 27


@pytest.fixture(scope='module')
def lib():
    return pq8.library()


def code(lib, name, *args):
    try:
        lib.call(name, *args)
    except pq8.PQ8Error as e:
        return e.code
    return 0


def rows(lib, x=X, kind=0, ld=64, q=Q, s=S, rows=4, width=64):
    return code(lib, 'pq8_quantize_rows', x, kind, ld, q, s, rows, width, None)


def test_quantize_rows_refusals(lib):
    assert rows(lib, rows=0) == 0
    assert rows(lib, rows=-1) == pq8.ERR_UNSUPPORTED_SHAPE
    for width in (0, -16, 8, 40, pq8.I8_MAX_K + 16):
        assert rows(lib, width=width, ld=1 << 18) == pq8.ERR_UNSUPPORTED_SHAPE, width
    assert rows(lib, kind=3) == pq8.ERR_INVALID_ARGUMENT
    assert rows(lib, ld=63) == pq8.ERR_INVALID_ARGUMENT
    assert rows(lib, x=None) == pq8.ERR_INVALID_ARGUMENT
    assert rows(lib, q=None) == pq8.ERR_INVALID_ARGUMENT
    assert rows(lib, s=None) == pq8.ERR_INVALID_ARGUMENT
    assert rows(lib, x=X + 2) == pq8.ERR_MISALIGNED
    assert rows(lib, x=X + 1, kind=1) == pq8.ERR_MISALIGNED
    assert rows(lib, q=Q + 8) == pq8.ERR_MISALIGNED
    assert rows(lib, s=S + 2) == pq8.ERR_MISALIGNED
    assert rows(lib, q=X + 64) == pq8.ERR_INVALID_ARGUMENT  # q inside x
    assert rows(lib, s=X + 64) == pq8.ERR_INVALID_ARGUMENT
    assert code(lib, 'pq8_layer_norm_quantize', X, 0, 64, None, B, Q, S, 4, 64, None) == pq8.ERR_INVALID_ARGUMENT
    assert code(lib, 'pq8_layer_norm_quantize', X, 0, 64, W, B + 1, Q, S, 4, 64, None) == pq8.ERR_MISALIGNED


def gemm(lib, w=W, ws=S, x=X, xs=S + 4096, y=Y, kind=0, bias=None, resid=None, m=4, n=64, k=64, epi=0):
    return code(lib, 'pq8_gemm_i8', w, ws, x, xs, y, kind, bias, resid, m, n, k, epi, 1.0, None)


def test_gemm_i8_refusals(lib):
    assert gemm(lib, m=0) == 0
    assert gemm(lib, m=-1) == pq8.ERR_UNSUPPORTED_SHAPE
    assert gemm(lib, n=0) == pq8.ERR_UNSUPPORTED_SHAPE
    for k in (0, 24, pq8.I8_MAX_K + 16):
        assert gemm(lib, k=k) == pq8.ERR_UNSUPPORTED_SHAPE, k
    assert gemm(lib, epi=5) == pq8.ERR_INVALID_ARGUMENT
    assert gemm(lib, epi=pq8.EPI_GLU, n=63) == pq8.ERR_UNSUPPORTED_SHAPE
    assert gemm(lib, epi=pq8.EPI_RESIDUAL) == pq8.ERR_INVALID_ARGUMENT  # no residual
    assert gemm(lib, kind=7) == pq8.ERR_INVALID_ARGUMENT
    for name in ('w', 'ws', 'x', 'xs', 'y'):
        assert gemm(lib, **{name: None}) == pq8.ERR_INVALID_ARGUMENT, name
    for name in ('w', 'x'):
        assert gemm(lib, **{name: {'w': W, 'x': X}[name] + 8}) == pq8.ERR_MISALIGNED
    assert gemm(lib, y=Y + 2) == pq8.ERR_MISALIGNED
    assert gemm(lib, y=Y + 1, kind=2) == pq8.ERR_MISALIGNED
    assert gemm(lib, bias=B + 2) == pq8.ERR_MISALIGNED
    for name, at in (('w', W + 64), ('x', X + 64), ('ws', S + 16), ('xs', S + 4096), ('bias', B)):
        kw = {'y': at}
        if name == 'bias':
            kw['bias'] = B
        assert gemm(lib, **kw) == pq8.ERR_INVALID_ARGUMENT, name
    # a residual that overlaps y without being y
    assert gemm(lib, epi=pq8.EPI_RESIDUAL, resid=Y + 64) == pq8.ERR_INVALID_ARGUMENT


def linear(lib, ld=64, kind=0, nw=None, nb=None, ws=WS, size=BIG, m=4, k=64, y=Y, x=X):
    return code(lib, 'pq8_linear_i8', W, S, x, kind, ld, nw, nb, y, 0, None, None, m, 64, k, 0, 1.0, ws, size, None)


def test_linear_i8_refusals(lib):
    need = lib.linear_i8_workspace_size(4, 64)
    assert need >= 4 * 64 + 16
    assert lib.linear_i8_workspace_size(0, 64) >= 0
    assert linear(lib, m=0, ws=None, size=0) == 0
    need = lib.linear_i8_workspace_size(9, 64)
    assert need == pq8.linear_i8_scratch(9, 64, 0) and pq8.linear_i8_scratch(8, 64, 0) == 0
    assert pq8.linear_i8_scratch(8, 1040, 0) == lib.linear_i8_workspace_size(8, 1040)
    assert pq8.linear_i8_scratch(1, 8192, 0) == 0 and pq8.linear_i8_scratch(1, 8208, 0) > 0
    assert pq8.linear_i8_scratch(2, 64, 8) == lib.linear_i8_workspace_size(2, 64)
    assert linear(lib, m=9, ws=None) == pq8.ERR_WORKSPACE
    assert linear(lib, m=9, size=need - 1) == pq8.ERR_WORKSPACE
    assert linear(lib, x=X + 4, ws=None) == pq8.ERR_WORKSPACE  # not the one-launch form
    assert linear(lib, ws=WS + 8) == pq8.ERR_MISALIGNED
    assert linear(lib, ld=60) == pq8.ERR_INVALID_ARGUMENT
    assert linear(lib, kind=-1) == pq8.ERR_INVALID_ARGUMENT
    assert linear(lib, nw=B) == pq8.ERR_INVALID_ARGUMENT  # weight without bias
    assert linear(lib, nb=B) == pq8.ERR_INVALID_ARGUMENT
    assert linear(lib, y=X + 128) == pq8.ERR_INVALID_ARGUMENT
    assert linear(lib, m=9, x=WS) == pq8.ERR_INVALID_ARGUMENT  # tokens inside the workspace
    assert linear(lib, m=9, y=WS + 64) == pq8.ERR_INVALID_ARGUMENT
    with pytest.raises(pq8.PQ8Error):
        lib.linear_i8_workspace_size(4, 65)
    assert code(lib, 'pq8_linear_i8_workspace_size', 4, 64, None) == pq8.ERR_INVALID_ARGUMENT


def norm(lib, x=X, kind=0, w=W, b=B, y=Y, rows=12, windows=3, off=None, c=64, g=4, eps=1e-5, act=0, flags=0, ws=WS,
         size=BIG):
    return code(lib, 'pq8_group_norm', x, kind, w, b, y, rows, windows, off, c, g, eps, act, flags, ws, size, None)


def test_group_norm_refusals(lib):
    assert norm(lib, rows=0) == 0
    assert norm(lib, rows=12, windows=0, off=S) == 0
    for kw in ({'rows': -1}, {'windows': -1}, {'rows': 13}, {'c': 0}, {'g': 0}, {'g': 5}, {'c': 16400, 'g': 1},
               {'c': 16384, 'g': 8192}, {'rows': (1 << 30) + 1, 'windows': 1}):
        assert norm(lib, **kw) == pq8.ERR_UNSUPPORTED_SHAPE, kw
    for kw in ({'kind': 4}, {'act': pq8.EPI_GLU}, {'act': pq8.EPI_RESIDUAL}, {'flags': 1}, {'kind': 1, 'flags': 2},
               {'eps': 0.0}, {'eps': -1.0}, {'eps': float('nan')}, {'eps': float('inf')}, {'x': None}, {'w': None},
               {'b': None}, {'y': None}, {'y': X}, {'y': X + 256}, {'y': W}, {'y': B}, {'off': Y}):
        assert norm(lib, **kw) == pq8.ERR_INVALID_ARGUMENT, kw
    for kw in ({'x': X + 2}, {'w': W + 2}, {'y': Y + 2}, {'y': Y + 1, 'kind': 2}, {'off': S + 2}, {'ws': WS + 8}):
        assert norm(lib, **kw) == pq8.ERR_MISALIGNED, kw
    assert lib.group_norm_workspace_size(0, 12, 3, 64, 4) == 0  # one launch
    need = lib.group_norm_workspace_size(0, 12, 3, 64, 4, quantize=True)
    assert need >= 3 * 4 * 16 and lib.group_norm_workspace_size(0, 12, 3, 64, 4, aligned16=False) > 0
    assert lib.group_norm_workspace_size(0, 0, 3, 64, 4) == lib.group_norm_workspace_size(0, 12, 0, 64, 4) == 0
    for bad in ((0, 12, 3, 64, 5), (3, 12, 3, 64, 4), (0, -1, 3, 64, 4)):
        with pytest.raises(pq8.PQ8Error):
            lib.group_norm_workspace_size(*bad)
    assert code(lib, 'pq8_group_norm_workspace_size', 0, 12, 3, 64, 4, 0, 0, 1, None) == pq8.ERR_INVALID_ARGUMENT
    assert code(lib, 'pq8_group_norm_quantize', X, 0, W, B, Q, S, 12, 3, None, 60, 4, 1e-5, 0, WS, BIG,
                None) == pq8.ERR_UNSUPPORTED_SHAPE
    assert code(lib, 'pq8_group_norm_quantize', X, 0, W, B, Q, None, 12, 3, None, 64, 4, 1e-5, 0, WS, BIG,
                None) == pq8.ERR_INVALID_ARGUMENT
    assert code(lib, 'pq8_group_norm_quantize', X, 0, W, B, Q + 8, S, 12, 3, None, 64, 4, 1e-5, 0, WS, BIG,
                None) == pq8.ERR_MISALIGNED
    assert code(lib, 'pq8_group_norm_quantize', X, 0, W, B, X, S, 12, 3, None, 64, 4, 1e-5, 0, WS, BIG,
                None) == pq8.ERR_INVALID_ARGUMENT


def test_oracle_quantize_ties_and_empty_rows():
    """The oracle itself: ties to even, a zero row, a row with an infinity."""
    h = np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 3.49, -3.51], [0.0] * 8, [np.inf] + [1.0] * 7])
    q, s, _ = oi.quantize(h)
    assert q[0].tolist() == [127, 0, 2, 2, 0, -2, 3, -4] and s[0] == 1.0
    assert not q[1].any() and s[1] == 0
    assert not q[2].any() and np.isnan(s[2])


def test_int8_refusals_at_the_edges(lib):
    """Sizes past 2^30, and outputs or workspaces inside what the call still has to read."""
    many = (1 << 30) + 1
    assert rows(lib, rows=many) == pq8.ERR_UNSUPPORTED_SHAPE
    assert gemm(lib, m=many) == gemm(lib, n=many) == pq8.ERR_UNSUPPORTED_SHAPE
    assert linear(lib, m=many) == pq8.ERR_UNSUPPORTED_SHAPE
    assert code(lib, 'pq8_linear_i8_workspace_size', many, 64, C.byref(C.c_size_t())) == pq8.ERR_UNSUPPORTED_SHAPE
    assert rows(lib, s=Q + 64) == pq8.ERR_INVALID_ARGUMENT  # scales inside q
    for q, s in ((W, S), (B, S), (Q, W), (Q, B)):
        assert code(lib, 'pq8_layer_norm_quantize', X, 0, 64, W, B, q, s, 4, 64, None) == pq8.ERR_INVALID_ARGUMENT
    assert linear(lib, y=B, nw=W + 64, nb=B) == pq8.ERR_INVALID_ARGUMENT  # y over the norm's bias
    for at in (W, S, B):  # the workspace over the weights, their scales, the norm
        assert linear(lib, m=9, ws=at, nw=B, nb=B + 4096) == pq8.ERR_INVALID_ARGUMENT, at
    for bias, resid in ((WS + 64, Y), (None, WS + 64)):
        assert code(lib, 'pq8_linear_i8', W, S, X, 0, 64, None, None, Y, 0, bias, resid, 9, 64, 64, pq8.EPI_RESIDUAL,
                    1.0, WS, BIG, None) == pq8.ERR_INVALID_ARGUMENT
    for eps in (9e-31, 1.1e30):
        assert norm(lib, eps=eps) == pq8.ERR_INVALID_ARGUMENT


def test_group_norm_workspace_sizes(lib):
    """The largest shapes that the size query takes: no size leaves 64 bits, none is missing."""
    for rows_, windows, c, g in ((1 << 30, 1, 16384, 4096), (1 << 30, 1, 16384, 1), (1 << 30, 1 << 24, 16, 16), (1, 1, 16, 16)):
        for quantize in (False, True):
            for ragged in (False, True):
                need = lib.group_norm_workspace_size(2, rows_, windows, c, g, ragged, quantize)
                assert 0 <= need < 1 << 48, (rows_, windows, c, g)
                assert need or not quantize


def test_int8_rows_whose_memory_is_of_another_type():
    """Integers or scales whose tensors were given memory of the same size but another type are refused."""
    import torch
    from parakeet_cuda_b200.runtime import Int8Weight
    q, s = torch.ones(32, 64, dtype=torch.int8), torch.ones(32)
    w8 = Int8Weight(q, s)
    assert w8.pointers() == (q.data_ptr(), s.data_ptr())
    for t, other in ((q, torch.ones(32, 16)), (s, torch.ones(32, dtype=torch.int32))):
        kept = t.data
        t.data = other
        with pytest.raises(ValueError):
            w8.pointers()
        t.data = kept
    assert w8.pointers() == (q.data_ptr(), s.data_ptr())


def test_gemm_i8_tile_refusals(lib):
    out = [C.byref(C.c_int()) for _ in range(3)]
    tile = lambda m=4, n=64, k=64, epi=0, out=out: code(lib, 'pq8_gemm_i8_tile', m, n, k, epi, *out)
    for kw in ({'m': 0}, {'m': -1}, {'m': (1 << 30) + 1}, {'n': 0}, {'k': 24}, {'k': pq8.I8_MAX_K + 16},
               {'epi': pq8.EPI_GLU, 'n': 63}):
        assert tile(**kw) == pq8.ERR_UNSUPPORTED_SHAPE, kw
    assert tile(epi=5) == pq8.ERR_INVALID_ARGUMENT
    for i in range(3):
        assert tile(out=out[:i] + [None] + out[i + 1:]) == pq8.ERR_INVALID_ARGUMENT
