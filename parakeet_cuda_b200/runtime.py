"""Host-side mirror of the reference's device runtime for the Q8_0 contraction path.

The reference keeps weights as GGUF Q8_0 bytes on the host, uploads a layer
at a time and expands it to FP32 with ``dequant_q8`` before every
``cublasSgemm_v2`` (``GPU.load_weights`` ``parakeet_cuda/gpu.py:169-184``,
``Blas.linear`` ``gpu.py:87-90``). Here the Q8_0 bytes are repacked once
(``pq8_pack_q8_0``), uploaded once and stay resident (all 24 encoder layers
are 642 MB), and every linear runs the fused library kernel on them.

``Runtime.load_weights(model, names)`` and ``Runtime.linear(...)`` keep the
reference's call shapes (``model`` is any object with ``gguf.Model``'s
``tensors``/``raw``/``array``). PyTorch is used only to own device memory and
streams; all arithmetic is in ``libpq8.so``.
"""
from __future__ import annotations

from dataclasses import dataclass
import ctypes as C
import warnings

import numpy as np
import torch

from . import pq8
from .pq8 import (EPI_GLU, EPI_NONE, GEMV_MAX_M, LAYOUT_GATES4, LAYOUT_GLU, LAYOUT_ROWS, TYPE_BF16,
                  TYPE_F16, TYPE_F32)

MIB = 1 << 20

# The current stream's handle by device index. torch.cuda.current_stream builds a Stream object
# around it, which costs as much as a launch.
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
# The current device's index, without the initialisation that torch.cuda.current_device looks for first.
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


@dataclass
class PackedWeight:
    """A resident packed Q8_0 tensor: ``n`` rows x ``k`` columns in ``layout``."""
    data: torch.Tensor  # uint8, device
    n: int
    k: int
    layout: int

    @property
    def pointer(self) -> int:
        return self.data.data_ptr()

    @property
    def out_features(self) -> int:
        return self.n // 2 if self.layout == LAYOUT_GLU else self.n // 4 if self.layout == LAYOUT_GATES4 else self.n


#: Element types of the 8-bit product's tokens and outputs and of the group norm.
ELEMENT_TYPES = {torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}


class _Int8Rows:
    """A dense int8 matrix with a float32 scale per row, checked once when it is made."""
    __slots__ = ('_q', '_scale', 'n', 'k', 'device', '_at')
    q = property(lambda self: self._q)
    scale = property(lambda self: self._scale)

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        if q.dtype != torch.int8 or q.dim() != 2 or not q.is_contiguous():
            raise ValueError(f'q must be a contiguous int8 matrix, got {q.dtype} {tuple(q.shape)}')
        if scale.dtype != torch.float32 or scale.dim() != 1 or not scale.is_contiguous():
            raise ValueError(f'scale must be a contiguous float32 vector, got {scale.dtype} {tuple(scale.shape)}')
        self.n, self.k = q.shape
        if scale.shape[0] != self.n:
            raise ValueError(f'{self.n} rows need {self.n} scales, got {scale.shape[0]}')
        self._at = q.get_device()
        if scale.get_device() != self._at:
            raise ValueError(f'q is on {q.device}, scale on {scale.device}')
        self._q, self._scale, self.device = q, scale, q.device

    def pointers(self) -> tuple[int, int]:
        """Addresses of the integers and the scales, as they are now (a tensor can be given other memory)."""
        q, scale = self._q, self._scale
        if (q.nbytes != self.n * self.k or scale.nbytes != 4 * self.n or q.dtype is not torch.int8
                or scale.dtype is not torch.float32 or q.get_device() != self._at or scale.get_device() != self._at
                or not (q.is_contiguous() and scale.is_contiguous())):
            raise ValueError('the integers or the scales have changed their size, type, layout or device')
        return q.data_ptr(), scale.data_ptr()


class Int8Weight(_Int8Rows):
    """Weights for the product in 8-bit integers: ``q`` int8 [n, k], ``scale`` float32 [n], one per output channel."""
    __slots__ = ()


class QuantizedRows(_Int8Rows):
    """Tokens quantised row by row: ``q`` int8 [rows, width], ``scale`` float32 [rows]; row i stands for
    ``q[i] * scale[i]``."""
    __slots__ = ()


def pack_host(raw, n: int, k: int, layout: int = LAYOUT_ROWS, lib=None) -> np.ndarray:
    """Repack GGUF Q8_0 bytes (``n*k/32`` x 34) into the packed format on the host."""
    lib = lib or pq8.library()
    raw = np.ascontiguousarray(raw, np.uint8)
    if raw.size != n * k // 32 * 34:
        raise ValueError(f'expected {n * k // 32 * 34} Q8_0 bytes for [{n}, {k}], got {raw.size}')
    out = np.empty(lib.packed_size(n, k, layout), np.uint8)
    lib.call('pq8_pack_q8_0', raw.ctypes.data, n, k, layout, out.ctypes.data)
    return out


def pack_concat_host(parts, n: int, layout: int, lib=None) -> np.ndarray:
    """Pack several ``[n, k_i]`` Q8_0 sources side by side along K (``parts = [(raw, k_i), ...]``)."""
    lib = lib or pq8.library()
    k_total = sum(k for _, k in parts)
    out = np.empty(lib.packed_size(n, k_total, layout), np.uint8)
    off = 0
    for raw, k in parts:
        raw = np.ascontiguousarray(raw, np.uint8)
        lib.call('pq8_pack_q8_0_part', raw.ctypes.data, n, k, k_total, off, layout, out.ctypes.data)
        off += k
    return out


def _host_bytes(raw) -> torch.Tensor:
    """A uint8 CPU tensor over ``raw``'s bytes (a GGUF memmap slice or any array), without a copy
    when ``raw`` is contiguous."""
    arr = np.ascontiguousarray(raw).reshape(-1).view(np.uint8)
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')  # read-only memmaps: the tensor is only ever read
        return torch.from_numpy(arr)


class _Slot:
    def __init__(self, nbytes: int, device, side: torch.cuda.Stream):
        self.host = torch.empty(nbytes, dtype=torch.uint8, pin_memory=True)
        self.dev = torch.empty(nbytes, dtype=torch.uint8, device=device)
        self.dev.record_stream(side)
        self.done = torch.cuda.Event()
        self.done.record(torch.cuda.current_stream(device))


class WeightUploader:
    """GGUF Q8_0 bytes -> resident packed weights, repacked on the device.

    Each tensor's raw bytes are copied (by torch's multi-threaded CPU copy)
    into one of two pinned staging buffers, sent to the device by an
    asynchronous copy on a side stream and repacked there by
    ``pq8_pack_q8_0_part_device``; meanwhile the host fills the other staging
    buffer. Nothing is packed or expanded on the host. This replaces the
    per-layer upload and ``dequant_q8`` of ``GPU.load_weights``
    (``parakeet_cuda/gpu.py:169-184``), which the reference repeats for every
    window. ``finish()`` makes the caller's stream wait for the uploads."""

    def __init__(self, runtime: 'Runtime', slot_bytes: int = 8 * MIB):
        self.rt = runtime
        self.side = torch.cuda.Stream(runtime.device)
        self.side.wait_stream(torch.cuda.current_stream(runtime.device))
        self.slots = [_Slot(slot_bytes, runtime.device, self.side) for _ in range(2)]
        self.turn = 0
        self.bytes_uploaded = 0

    def _slot(self, nbytes: int) -> _Slot:
        slot = self.slots[self.turn]
        self.turn ^= 1
        slot.done.synchronize()  # its previous copy and repack have finished reading it
        if slot.host.numel() < nbytes:
            self.slots[self.turn ^ 1] = slot = _Slot(max(nbytes, 2 * slot.host.numel()), self.rt.device, self.side)
            self.side.wait_stream(torch.cuda.current_stream(self.rt.device))
        return slot

    def _stage(self, raws) -> tuple[_Slot, int]:
        """Copy ``raws`` back to back into a staging buffer and start its upload."""
        srcs = [_host_bytes(r) for r in raws]
        nbytes = sum(t.numel() for t in srcs)
        slot = self._slot(nbytes)
        off = 0
        for t in srcs:  # torch's CPU copy (threaded for large tensors) into pinned memory
            slot.host[off:off + t.numel()].copy_(t)
            off += t.numel()
        with torch.cuda.stream(self.side):
            slot.dev[:nbytes].copy_(slot.host[:nbytes], non_blocking=True)
        self.bytes_uploaded += nbytes
        return slot, nbytes

    def _output(self, nbytes: int) -> torch.Tensor:
        # allocated for the caller's stream, written on the side stream
        out = torch.empty(nbytes, dtype=torch.uint8, device=self.rt.device)
        self.side.wait_stream(torch.cuda.current_stream(self.rt.device))
        out.record_stream(self.side)
        return out

    def pack(self, parts, n: int, layout: int = LAYOUT_ROWS) -> PackedWeight:
        """``parts = [(raw, k_i), ...]``: GGUF Q8_0 ``[n, k_i]`` sources packed side by side along K."""
        lib = self.rt.lib
        k_total = sum(k for _, k in parts)
        packed = self._output(lib.packed_size(n, k_total, layout))
        off = 0
        for raw, k in parts:
            slot, nbytes = self._stage([raw])
            if nbytes != n * k // 32 * 34:
                raise ValueError(f'expected {n * k // 32 * 34} Q8_0 bytes for [{n}, {k}], got {nbytes}')
            with torch.cuda.stream(self.side):
                lib.call('pq8_pack_q8_0_part_device', slot.dev.data_ptr(), n, k, k_total, off, layout,
                         packed.data_ptr(), C.c_void_p(self.side.cuda_stream))
                slot.done.record(self.side)
            off += k
        return PackedWeight(packed, n, k_total, layout)

    def pack_rows(self, raws, n: int, k: int, layout: int = LAYOUT_ROWS) -> PackedWeight:
        """GGUF Q8_0 sources stacked along N (e.g. Q, K, V into one [3n', k] matrix)."""
        lib = self.rt.lib
        packed = self._output(lib.packed_size(n, k, layout))
        slot, nbytes = self._stage(raws)
        if nbytes != n * k // 32 * 34:
            raise ValueError(f'expected {n * k // 32 * 34} Q8_0 bytes for [{n}, {k}], got {nbytes}')
        with torch.cuda.stream(self.side):
            lib.call('pq8_pack_q8_0_device', slot.dev.data_ptr(), n, k, layout, packed.data_ptr(),
                     C.c_void_p(self.side.cuda_stream))
            slot.done.record(self.side)
        return PackedWeight(packed, n, k, layout)

    def finish(self) -> None:
        torch.cuda.current_stream(self.rt.device).wait_stream(self.side)


class Runtime:
    """One device's resident weights, workspace and launch helpers."""

    def __init__(self, device: int | torch.device = 0, workspace_bytes: int = 8 * MIB):
        if not torch.cuda.is_available():
            raise RuntimeError('pq8 needs a CUDA device (B200, sm_100a); no CPU fallback exists')
        self.device = torch.device('cuda', device) if isinstance(device, int) else torch.device(device)
        if self.device.index is None:
            self.device = torch.device('cuda', torch.cuda.current_device())
        self.lib = pq8.library()
        with torch.cuda.device(self.device):
            self.workspace = torch.empty(workspace_bytes, dtype=torch.uint8, device=self.device)
            self.lib.call('pq8_workspace_init', self.workspace.data_ptr(), workspace_bytes, self.stream())
        self.weights: dict[str, object] = {}
        self._uploader: WeightUploader | None = None

    # -- plumbing ---------------------------------------------------------
    def stream(self):
        return C.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)

    def upload_packed(self, packed: np.ndarray, n: int, k: int, layout: int) -> PackedWeight:
        host = torch.from_numpy(np.ascontiguousarray(packed))
        return PackedWeight(host.to(self.device, non_blocking=False), n, k, layout)

    def uploader(self) -> WeightUploader:
        if self._uploader is None:
            self._uploader = WeightUploader(self)
        return self._uploader

    def pack(self, raw, n: int, k: int, layout: int = LAYOUT_ROWS) -> PackedWeight:
        """Resident packed copy of GGUF Q8_0 bytes ``raw`` ([n, k]), repacked on the device."""
        up = self.uploader()
        w = up.pack([(raw, k)], n, layout)
        up.finish()
        return w

    # -- GPU.load_weights counterpart ---------------------------------------
    def load_weights(self, model, names, layouts: dict | None = None) -> dict:
        """Upload tensors once and keep them resident.

        Q8_0 tensors are repacked (``layouts[name]`` selects GLU pairing);
        F32 tensors become float32 device tensors; F16 tensors stay fp16.
        """
        layouts = layouts or {}
        up = self.uploader()
        for name in names:
            t = model.tensors[name]
            if t.kind == 8:
                n, k = t.shape[0], int(np.prod(t.shape[1:]))
                self.weights[name] = up.pack([(model.raw(name), k)], n, layouts.get(name, LAYOUT_ROWS))
            elif t.kind == 1:
                self.weights[name] = torch.from_numpy(np.ascontiguousarray(model.raw(name)).view(np.float16).copy()
                                                      ).reshape(t.shape).to(self.device)
            else:
                self.weights[name] = torch.from_numpy(np.ascontiguousarray(model.raw(name)).view(np.float32).copy()
                                                      ).reshape(t.shape).to(self.device)
        up.finish()
        return self.weights

    def weight(self, name):
        return self.weights[name]

    # -- workspace ----------------------------------------------------------
    def ensure_workspace(self, m: int, n: int, k: int) -> None:
        need = self.lib.linear_workspace_size(m, n, k)
        if need > self.workspace.numel():
            with torch.cuda.device(self.device):
                self.workspace = torch.empty(max(need, 2 * self.workspace.numel()), dtype=torch.uint8,
                                             device=self.device)
                self.lib.call('pq8_workspace_init', self.workspace.data_ptr(), self.workspace.numel(), self.stream())

    # -- Blas.linear counterpart ---------------------------------------------
    def linear(self, x: torch.Tensor, w: PackedWeight, out: torch.Tensor | None = None, bias=None, resid=None,
               epilogue: int = EPI_NONE, alpha: float = 1.0, flags: int = 0) -> torch.Tensor:
        """``out = epilogue(x @ W^T + bias)`` for a resident packed ``w`` (any number of rows)."""
        rows, k = x.shape
        if k != w.k:
            raise ValueError(f'x has {k} columns, weight has {w.k}')
        if out is None:
            out = torch.empty(rows, w.out_features if epilogue == EPI_GLU else w.n, dtype=torch.float32,
                              device=self.device)
        if rows >= 1:
            self.ensure_workspace(rows, w.n, k)
        self.lib.call('pq8_linear', w.pointer, x.data_ptr(), out.data_ptr(), _ptr(bias), _ptr(resid), rows, w.n, k,
                      epilogue, float(alpha), flags, self.workspace.data_ptr(), self.workspace.numel(),
                      self.stream())
        return out

    def gemm(self, x, w: PackedWeight, out=None, bias=None, resid=None, epilogue=EPI_NONE, alpha=1.0, flags=0):
        """Always the tensor-core kernel (any m), regardless of the GEMV dispatch threshold."""
        rows, k = x.shape
        if out is None:
            out = torch.empty(rows, w.out_features if epilogue == EPI_GLU else w.n, dtype=torch.float32,
                              device=self.device)
        self.lib.call('pq8_gemm', w.pointer, x.data_ptr(), out.data_ptr(), _ptr(bias), _ptr(resid), rows, w.n, k,
                      epilogue, float(alpha), flags, self.stream())
        return out

    # -- products in 8-bit integers -------------------------------------------
    # These calls take a few microseconds of GPU time for a few tokens, so the
    # host path is kept short: each tensor is checked once, and outputs are
    # allocated by the cheapest call torch has for it.
    def _check(self, t: torch.Tensor, what: str, dtype, shape) -> int:
        """Address of a dense tensor of ``dtype`` and ``shape`` on this device."""
        if t.dtype is not dtype or t.shape != shape or t.get_device() != self.device.index or not t.is_contiguous():
            raise ValueError(f'{what} must be contiguous {dtype} {tuple(shape)} on {self.device}, got '
                             f'{"" if t.is_contiguous() else "strided "}{t.dtype} {tuple(t.shape)} on {t.device}')
        return t.data_ptr()

    def _check_rows(self, x: torch.Tensor) -> tuple[int, int, int, int]:
        """(rows, width, row distance, type code) of a matrix whose rows are dense."""
        kind = ELEMENT_TYPES.get(x.dtype)
        if kind is None or x.dim() != 2 or x.get_device() != self.device.index:
            raise ValueError(f'x must be a float32, float16 or bfloat16 matrix on {self.device}, got {x.dtype} '
                             f'{tuple(x.shape)} on {x.device}')
        rows, width = x.shape
        if rows > 1 << 30:
            raise ValueError(f'at most 2^30 rows a call, got {rows}')
        ld, step = x.stride()
        if rows <= 1:
            ld = width
        if (step != 1 and width > 1) or ld < width:
            raise ValueError(f'the rows of x must be dense and apart, got strides {x.stride()}')
        return rows, width, ld, kind

    def _enqueue(self, call: str, *args) -> None:
        """A library call on this device's current stream."""
        index = self.device.index
        args += (_raw_stream(index),)
        if _current_device() == index:
            code = getattr(self.lib.lib, call)(*args)
        else:
            with torch.cuda.device(index):
                code = getattr(self.lib.lib, call)(*args)
        if code:
            raise pq8.PQ8Error(call, code, self.lib.error_string(code))

    def _new_rows(self, rows: int, width: int) -> tuple[QuantizedRows, int, int]:
        """Rows to be written, and the addresses of their integers and scales."""
        q = torch.empty(rows, width, dtype=torch.int8, device=self.device)
        scale = torch.empty(rows, dtype=torch.float32, device=self.device)
        return QuantizedRows(q, scale), q.data_ptr(), scale.data_ptr()

    def quantize_rows(self, x: torch.Tensor, norm=None) -> QuantizedRows:
        """``x`` [rows, width] (float32, float16 or bfloat16; rows dense, any row distance) to 8-bit
        integers with one scale per row, ``norm=(weight, bias)`` applying LayerNorm first. The
        integers are those of the exact quotient (ties to even); ``width`` a multiple of 16."""
        rows, width, ld, kind = self._check_rows(x)
        out, q, scale = self._new_rows(rows, width)
        if norm is None:
            self._enqueue('pq8_quantize_rows', x.data_ptr(), kind, ld, q, scale, rows, width)
        else:
            w = self._check(norm[0], 'the norm weight', torch.float32, (width,))
            b = self._check(norm[1], 'the norm bias', torch.float32, (width,))
            self._enqueue('pq8_layer_norm_quantize', x.data_ptr(), kind, ld, w, b, q, scale, rows, width)
        return out

    def int8_weight(self, w) -> Int8Weight:
        """Weights [n, k] (a float tensor, or a ``(raw, n, k)`` triple of GGUF Q8_0 bytes and its shape)
        quantised to 8 bits with one scale per output channel."""
        if isinstance(w, tuple):
            raw, n, k = w
            if k % 32:
                raise ValueError(f'a Q8_0 row is whole blocks of 32, got {k} columns')
            blocks = _host_bytes(raw).to(self.device)
            if blocks.numel() != n * k // 32 * 34:
                raise ValueError(f'expected {n * k // 32 * 34} Q8_0 bytes for [{n}, {k}], got {blocks.numel()}')
            w = torch.empty(n, k, dtype=torch.float32, device=self.device)
            self._enqueue('pq8_dequant_q8_0', blocks.data_ptr(), w.data_ptr(), n * k)
        rows = self.quantize_rows(w)
        return Int8Weight(rows.q, rows.scale)

    def linear_i8(self, x, w: Int8Weight, out: torch.Tensor | None = None, bias=None, resid=None,
                  epilogue: int = EPI_NONE, alpha: float = 1.0, norm=None, out_dtype=None) -> torch.Tensor:
        """``out = epilogue((x @ W^T) + bias)`` with the product in 8-bit integers.

        ``x``: float tokens [rows, k], quantised per row on the way (after a LayerNorm with
        ``norm=(weight, bias)``), or ``QuantizedRows``. Epilogues as ``linear``; ``EPI_GLU`` takes the
        plain rows of ``w`` (gates in the second half). ``out_dtype``: float32 (the default),
        float16 or bfloat16; ``out``, ``resid`` have it. ``out`` may be ``resid``, no other input."""
        device = self.device
        if type(w) is not Int8Weight or w._at != device.index:
            raise ValueError(f'the weight must be an Int8Weight on {device}')
        n, k = w.n, w.k
        quantized = type(x) is QuantizedRows
        if quantized:
            rows, width = x.n, x.k
            if norm is not None:
                raise ValueError('quantised tokens take no norm')
            if x._at != device.index:
                raise ValueError(f'x is on {x.device}, the runtime on {device}')
        else:
            rows, width, ld, kind = self._check_rows(x)
        if width != k:
            raise ValueError(f'x has {width} columns, weight has {k}')
        cols = n // 2 if epilogue == EPI_GLU else n
        if out is None:
            out = torch.empty(rows, cols, dtype=out_dtype or torch.float32, device=device)
            y = out.data_ptr()
        else:
            y = self._check(out, 'out', out_dtype or out.dtype, (rows, cols))
        y_kind = ELEMENT_TYPES.get(out.dtype)
        if y_kind is None:
            raise ValueError(f'the output must be float32, float16 or bfloat16, got {out.dtype}')
        b = None if bias is None else self._check(bias, 'bias', torch.float32, (n,))
        r = None if resid is None else self._check(resid, 'resid', out.dtype, (rows, cols))
        if quantized:
            self._enqueue('pq8_gemm_i8', *w.pointers(), *x.pointers(), y, y_kind, b, r, rows, n, k, epilogue, alpha)
            return out
        g = h = None
        if norm is not None:
            g = self._check(norm[0], 'the norm weight', torch.float32, (k,))
            h = self._check(norm[1], 'the norm bias', torch.float32, (k,))
        # scratch of this call alone: calls on other streams and captured graphs have their own
        at = x.data_ptr()
        need = pq8.linear_i8_scratch(rows, k, at | (0 if rows <= 1 else ld * x.element_size()) | (g or 0) | (h or 0))
        scratch = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        self._enqueue('pq8_linear_i8', *w.pointers(), at, kind, ld, g, h, y, y_kind, b, r, rows, n, k,
                      epilogue, alpha, _ptr(scratch), need)
        return out

    # -- group norm --------------------------------------------------------------
    def _check_group_norm(self, x, weight, bias, groups, windows, offsets):
        """(rows, channels, type code, addresses of x, weight, bias and offsets)."""
        kind = ELEMENT_TYPES.get(x.dtype)
        if kind is None or x.dim() != 2:
            raise ValueError(f'x must be a float32, float16 or bfloat16 matrix, got {x.dtype} {tuple(x.shape)}')
        rows, channels = x.shape
        if rows > 1 << 30 or not 0 < groups <= channels or windows > 1 << 24:
            raise ValueError(f'{rows} rows in {windows} windows, {channels} channels in {groups} groups: at most 2^30 rows '
                             'in 2^24 windows, and a group has a channel')
        at = (self._check(x, 'x', x.dtype, x.shape), self._check(weight, 'weight', torch.float32, (channels,)),
              self._check(bias, 'bias', torch.float32, (channels,)))
        off = None
        if offsets is not None:
            off = self._check(offsets, 'offsets', torch.int32, (windows + 1,))
        elif windows < 1 or rows % windows:
            raise ValueError(f'{rows} rows do not make {windows} windows of equal length')
        return rows, channels, kind, at, off

    def group_norm(self, x: torch.Tensor, weight, bias, groups: int, windows: int = 1, offsets=None,
                   eps: float = 1e-5, epilogue: int = EPI_NONE, flags: int = 0,
                   out: torch.Tensor | None = None) -> torch.Tensor:
        """Group norm and activation (``EPI_NONE``, ``EPI_RELU`` or ``EPI_SILU``), channels last: ``x``
        [rows, channels] in ``windows`` windows of equal length, or of the rows ``offsets[i]`` to
        ``offsets[i + 1] - 1`` (int32 on the device, ``windows + 1`` of them). Rows in no window are
        not written: ``out`` keeps what it held, and a new tensor has nothing there."""
        rows, channels, kind, at, off = self._check_group_norm(x, weight, bias, groups, windows, offsets)
        if out is None:
            out = torch.empty_like(x)
            y = out.data_ptr()
        else:
            y = self._check(out, 'out', x.dtype, x.shape)
        need = self.lib.group_norm_workspace_size(kind, rows, windows, channels, groups, off is not None, False,
                                                  not (at[0] | y) & 15)
        scratch = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._enqueue('pq8_group_norm', at[0], kind, at[1], at[2], y, rows, windows, off, channels, groups, eps,
                      epilogue, flags, _ptr(scratch), need)
        return out

    def group_norm_quantize(self, x: torch.Tensor, weight, bias, groups: int, windows: int = 1, offsets=None,
                            eps: float = 1e-5, epilogue: int = EPI_NONE) -> QuantizedRows:
        """``group_norm``, its rows quantised as ``quantize_rows`` does, for ``linear_i8``. Rows in no window
        are zeros with scale 0: a ``linear_i8`` that follows leaves their residual as it is."""
        rows, channels, kind, at, off = self._check_group_norm(x, weight, bias, groups, windows, offsets)
        out, q, scale = self._new_rows(rows, channels)
        need = self.lib.group_norm_workspace_size(kind, rows, windows, channels, groups, off is not None, True,
                                                  not (at[0] | at[1] | at[2]) & 15)
        scratch = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._enqueue('pq8_group_norm_quantize', at[0], kind, at[1], at[2], q, scale, rows, windows, off,
                      channels, groups, eps, epilogue, _ptr(scratch), need)
        return out

    def device_status(self) -> int:
        return self.lib.device_status(self.stream())
