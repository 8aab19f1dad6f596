"""The 8-bit operators on torch tensors: e4m3 rows with one f32 scale per row and 128 columns.

add_norm_f8 writes such rows (svl_add_norm_f8_device), F8Linear multiplies them by an e4m3 matrix
with a scale per 128 x 128 block (svl_f8_linear_device). Both enqueue on torch's current stream of
the tensors' device, or on `stream`, and may be captured into CUDA graphs.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from .model import tensor_views

BLOCK = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_NORMS = {None: -1, "layer": 0, "rms": 1}


def _rows(name: str, t, shape=None, dtypes=_DTYPES):
    """Checks a [rows][columns] CUDA tensor whose columns are contiguous."""
    if t.dim() != 2 or not t.is_cuda or t.dtype not in dtypes or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be a CUDA tensor [rows, columns] with contiguous columns, of "
                         f"{', '.join(str(d) for d in dtypes)}: got {tuple(t.shape)}, {t.dtype}, {t.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}: got {tuple(t.shape)}")


def _row_stride(t) -> int:
    """Elements between a tensor's rows (torch leaves a single row's stride undefined)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _vector(name: str, t, n: int, device):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be {n} contiguous float32 values on {device}: got {tuple(t.shape)}, {t.dtype}, {t.device}")
    return t.data_ptr()


def _stream(stream, device):
    return (torch.cuda.current_stream(device) if stream is None else stream).cuda_stream


def add_norm_f8(x, residual=None, norm: str | None = "rms", weight=None, bias=None, eps: float = 1e-8,
                out_sum=None, stream=None):
    """h = x + residual, y = norm(h) ("rms", "layer" or None: y = h), y as e4m3 rows.

    x and residual: CUDA [rows, k], float32 or bfloat16; weight and bias: float32 [k] or None.
    Returns (q, scales, h): q float8_e4m3fn [rows, k] (rows 16-byte aligned), scales float32
    [ceil(k / 128), rows], and the sum h in x's dtype: out_sum if given (it may be x or residual),
    a new tensor with a residual, x itself without."""
    _rows("x", x)
    rows, k = x.shape
    device = x.device
    if norm not in _NORMS:
        raise ValueError(f"norm must be 'rms', 'layer' or None: got {norm!r}")
    for name, t in (("residual", residual), ("out_sum", out_sum)):
        if t is not None:
            _rows(name, t, x.shape, (x.dtype,))
            if t.device != device:
                raise ValueError(f"{name} is on {t.device}, x on {device}")
    w, b = _vector("weight", weight, k, device), _vector("bias", bias, k, device)
    h = out_sum if out_sum is not None else x if residual is None else torch.empty((rows, k), dtype=x.dtype, device=device)
    ld = (k + 15) // 16 * 16
    q = torch.empty((rows, ld), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty(((k + BLOCK - 1) // BLOCK, rows), dtype=torch.float32, device=device)
    keep = h is not x
    _lib.check(_lib.lib().svl_add_norm_f8_device(
        device.index, rows, k, _DTYPES[x.dtype], x.data_ptr(), _row_stride(x),
        None if residual is None else residual.data_ptr(), 0 if residual is None else _row_stride(residual),
        _NORMS[norm], w, b, eps, h.data_ptr() if keep or residual is not None else None, _row_stride(h), q.data_ptr(), ld,
        scales.data_ptr(), rows, _stream(stream, device)))
    return q[:, :k] if ld != k else q, scales, h


class F8Linear:
    """An e4m3 matrix [n][k] with f32 scales per 128 x 128 block, and an optional bias.

    weight: float8_e4m3fn CUDA [n, k], scales: float32 CUDA [ceil(n / 128), ceil(k / 128)], bias:
    float32 CUDA [n] or None; all are copied. F8Linear.quantise() makes one from f32 weights."""

    handle = None

    def __init__(self, weight, scales, bias=None, stream=None):
        _rows("weight", weight, dtypes=(torch.float8_e4m3fn,))
        n, k = weight.shape
        device = weight.device
        blocks = ((n + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK)
        _rows("scales", scales, blocks, (torch.float32,))
        s, b = _vector("scales", scales, blocks[0] * blocks[1], device), _vector("bias", bias, n, device)
        h = ctypes.c_void_p()
        _lib.check(_lib.lib().svl_f8_linear_create_device(n, k, weight.data_ptr(), _row_stride(weight), s, b, device.index,
                                                          _stream(stream, device), ctypes.byref(h)))
        self._set(h, n, k, device)

    @classmethod
    def quantise(cls, weight: np.ndarray, bias: np.ndarray | None = None, device: int = 0) -> "F8Linear":
        """From host f32 weights [n][k] (and a bias [n]): each block's scale is its largest
        magnitude / 448."""
        tensors = {"weight": weight} if bias is None else {"weight": weight, "bias": bias}
        views, keep = tensor_views(tensors)
        h = ctypes.c_void_p()
        _lib.check(_lib.lib().svl_f8_linear_create(weight.shape[0], weight.shape[1], views, len(tensors), device,
                                                   ctypes.byref(h)))
        del keep
        self = cls.__new__(cls)
        self._set(h, weight.shape[0], weight.shape[1], torch.device("cuda", device))
        return self

    def _set(self, handle, n: int, k: int, device):
        self.handle, self.n, self.k, self.device = handle, n, k, device
        # Bound now: at interpreter exit the module globals may already be gone.
        self._destroy = _lib.lib().svl_f8_linear_destroy

    def __call__(self, q, scales, out_dtype=torch.float32, out=None, stream=None):
        """q: float8_e4m3fn CUDA [rows, k], 16-byte aligned rows, scales: float32 [ceil(k / 128),
        rows] (both as add_norm_f8 returns them) -> [rows, n] of out_dtype, in `out` if given."""
        rows = q.shape[0]
        _rows("q", q, (rows, self.k), (torch.float8_e4m3fn,))
        _rows("scales", scales, ((self.k + BLOCK - 1) // BLOCK, rows), (torch.float32,))
        if q.device != self.device or scales.device != self.device:
            raise ValueError(f"q and scales must be on {self.device}")
        if out is None:
            out = torch.empty((rows, self.n), dtype=out_dtype, device=self.device)
        _rows("out", out, (rows, self.n))
        if out.device != self.device:
            raise ValueError(f"out must be on {self.device}")
        ld = q.stride(0) if rows > 1 else (self.k + 15) // 16 * 16  # a single row's stride is never used
        _lib.check(_lib.lib().svl_f8_linear_device(self.handle, rows, q.data_ptr(), ld, scales.data_ptr(),
                                                   _row_stride(scales), _DTYPES[out.dtype], out.data_ptr(), _row_stride(out),
                                                   _stream(stream, self.device)))
        return out

    def check(self):
        """Waits for the device; raises if a bounded device-side wait of a product ran out."""
        _lib.check(_lib.lib().svl_f8_linear_error(self.handle))

    def close(self):
        if self.handle:
            self._destroy(self.handle)
            self.handle = None

    __del__ = close
