"""The 8-bit operators on torch tensors: e4m3 rows with one f32 scale per row and 128 columns.

add_norm_f8 writes such rows (svl_add_norm_f8_device), F8Linear multiplies them by an e4m3 matrix
with a scale per 128 x 128 block (svl_f8_linear_device). Both enqueue on torch's current stream of
the tensors' device, or on `stream`, and may be captured into CUDA graphs. They are for inference: inputs that
require a gradient are taken, but outputs are detached from them.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from ._ops import of, on, ops
from .model import tensor_views

BLOCK = 128
_NORMS = {None: -1, "layer": 0, "rms": 1}


def add_norm_f8(x, residual=None, norm: str | None = "rms", weight=None, bias=None, eps: float = 1e-8,
                out_sum=None, stream=None):
    """h = x + residual, y = norm(h) ("rms", "layer" or None: y = h), y as e4m3 rows.

    x and residual: CUDA [rows, k], float32 or bfloat16; weight (of a norm) and bias (of the layer norm):
    float32 [k] or None.
    Returns (q, scales, h): q float8_e4m3fn [rows, k] (rows 16-byte aligned), scales float32
    [ceil(k / 128), rows], and the sum h in x's dtype: out_sum if given (it may be x or residual),
    a new tensor with a residual, x itself without. out_sum must not overlap x or residual otherwise."""
    if stream is not None:
        with on(stream, x.device):
            return add_norm_f8(x, residual, norm, weight, bias, eps, out_sum)
    kind = _NORMS.get(norm, 2)  # 2: refused by name below the binding
    return ops.add_norm_f8(x, residual, kind, weight, bias, eps, out_sum)


class F8Linear:
    """An e4m3 matrix [n][k] with f32 scales per 128 x 128 block, and an optional bias.

    weight: float8_e4m3fn CUDA [n, k], scales: float32 CUDA [ceil(n / 128), ceil(k / 128)], bias:
    float32 CUDA [n] or None; all are copied, after the work on torch's current stream of their device (or on
    `stream`), which the call waits for. F8Linear.quantise() makes one from f32 weights. It has to outlive the
    CUDA graphs that captured its products."""

    handle = None

    def __init__(self, weight, scales, bias=None, stream=None):
        if not weight.is_cuda or weight.dim() != 2 or weight.dtype != torch.float8_e4m3fn or \
                (weight.shape[1] > 1 and weight.stride(1) != 1):
            raise ValueError("weight must be a CUDA tensor [n, k] of float8_e4m3fn with contiguous columns: "
                             f"got {tuple(weight.shape)}, {weight.dtype}, {weight.device}")
        n, k = weight.shape
        device = weight.device
        blocks = ((n + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK)
        for name, t, shape in (("scales", scales, blocks), ("bias", bias, (n,))):
            if t is not None and (tuple(t.shape) != shape or t.dtype != torch.float32 or not t.is_contiguous() or t.device != device):
                raise ValueError(f"{name} must be contiguous float32 {shape} on {device}: got {tuple(t.shape)}, {t.dtype}, {t.device}")
        h = ctypes.c_void_p()
        s = torch.cuda.current_stream(device) if stream is None else of(stream, device)
        _lib.check(_lib.lib().svl_f8_linear_create_device(
            n, k, weight.data_ptr(), weight.stride(0) if n > 1 else max(weight.stride(0), k), scales.data_ptr(),
            None if bias is None else bias.data_ptr(), device.index, s.cuda_stream, ctypes.byref(h)))
        self._set(h, n, k, device.index)

    @classmethod
    def quantise(cls, weight: np.ndarray, bias: np.ndarray | None = None, device: int = 0) -> "F8Linear":
        """From host f32 weights [n][k] (and a bias [n]): each block's scale is its largest
        magnitude / 448."""
        n, k = weight.shape
        tensors = {"weight": weight} if bias is None else {"weight": weight, "bias": bias}
        views, keep = tensor_views(tensors)
        h = ctypes.c_void_p()
        _lib.check(_lib.lib().svl_f8_linear_create(n, k, views, len(tensors), device, ctypes.byref(h)))
        del keep
        self = cls.__new__(cls)
        self._set(h, n, k, device)
        return self

    def _set(self, handle, n: int, k: int, device: int):
        self.handle, self.n, self.k, self.device = handle.value, n, k, device
        # Bound now: at interpreter exit the module globals may already be gone.
        self._destroy = _lib.lib().svl_f8_linear_destroy

    def __call__(self, q, scales, out_dtype=torch.float32, out=None, stream=None):
        """q: float8_e4m3fn CUDA [rows, k], 16-byte aligned rows, scales: float32 [ceil(k / 128),
        rows] (both as add_norm_f8 returns them) -> [rows, n] of out_dtype, or `out` (whose dtype
        counts then). The call does not wait: if a bounded wait of the product on the device ran out, only
        check() tells, and the outputs are undefined."""
        if self.handle is None:
            raise ValueError("the F8Linear is closed")
        if stream is not None:
            with on(stream, torch.device("cuda", self.device)):
                return self(q, scales, out_dtype, out)
        return ops.f8_linear(self.handle, self.n, self.k, self.device, q, scales, out_dtype, out)

    def __reduce_ex__(self, protocol):
        # A copy would own the same matrix, and both would free it.
        raise TypeError("an F8Linear cannot be copied or pickled")

    def check(self):
        """Waits for the device; raises if a bounded device-side wait of a product ran out."""
        _lib.check(_lib.lib().svl_f8_linear_error(self.handle))

    def close(self):
        if self.handle:
            self._destroy(self.handle)
            self.handle = None

    __del__ = close
