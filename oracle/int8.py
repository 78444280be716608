"""64-bit oracle of the 8-bit product, the row quantisation and the group norm
(NumPy; written from their definitions in include/pq8.h)."""
from __future__ import annotations

import numpy as np

EPS = 1e-5


def quantize(h):
    """(q, scale, margin) of rows ``h`` (float64 values): scale = max|h| / 127 rounded to fp32, q the
    nearest integer to h / scale (ties to even), margin the distance of each quotient to the nearest
    border between two integers. Rows with an infinity or a NaN: scale NaN, q 0."""
    h = np.asarray(h, np.float64)
    top = np.abs(h).max(axis=1)
    fine = np.isfinite(top)
    scale = np.where(fine, top, 0.0) / 127.0
    scale = scale.astype(np.float32)
    s = scale.astype(np.float64)[:, None]
    with np.errstate(all='ignore'):
        u = np.where(s > 0, h / np.where(s > 0, s, 1.0), 0.0)
    u = np.where(fine[:, None], u, 0.0)
    q = np.clip(np.rint(u), -127, 127).astype(np.int8)
    margin = np.abs(np.abs(u - np.floor(u)) - 0.5)
    return q, np.where(fine, scale, np.float32(np.nan)).astype(np.float32), margin


def layer_norm(x, w, b, eps=EPS):
    x = np.asarray(x, np.float64)
    mean = x.mean(axis=1, keepdims=True)
    var = ((x - mean) ** 2).mean(axis=1, keepdims=True)
    return (x - mean) / np.sqrt(var + eps) * np.asarray(w, np.float64) + np.asarray(b, np.float64)


def sigmoid(z):
    with np.errstate(over='ignore'):
        return 1.0 / (1.0 + np.exp(-z))


def act(z, name):
    return np.maximum(z, 0) if name == 'relu' else z * sigmoid(z) if name == 'silu' else z


def product(q, s, w, t, bias=None):
    """(z, size): the scaled integer product plus bias in float64, and the sum of its terms' magnitudes
    (what its fp32 roundings are relative to). Integer sums in int64."""
    acc = q.astype(np.int64) @ w.astype(np.int64).T
    p = acc.astype(np.float64) * np.asarray(s, np.float64)[:, None] * np.asarray(t, np.float64)[None, :]
    b = 0.0 if bias is None else np.asarray(bias, np.float64)[None, :]
    return p + b, np.abs(p) + np.abs(b)


def group_norm(x, w, b, groups, bounds, eps=EPS, epilogue='none'):
    """Rows of no window are NaN."""
    x = np.asarray(x, np.float64)
    out = np.full(x.shape, np.nan)
    c = x.shape[1]
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        if hi <= lo:
            continue
        blk = x[lo:hi].reshape(hi - lo, groups, c // groups)
        mean = blk.mean(axis=(0, 2), keepdims=True)
        var = ((blk - mean) ** 2).mean(axis=(0, 2), keepdims=True)
        z = ((blk - mean) / np.sqrt(var + eps)).reshape(hi - lo, c)
        out[lo:hi] = act(z * np.asarray(w, np.float64) + np.asarray(b, np.float64), epilogue)
    return out
