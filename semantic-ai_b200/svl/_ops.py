"""The operators' binding to torch tensors (csrc/torch_ops.cpp): checks, output tensors and the
current stream in C++, around the C ABI that _lib loads."""
from __future__ import annotations

import ctypes

import torch  # the binding's symbols too

from . import _lib

try:
    from . import _torch_ops as ops
except ImportError as e:
    raise ImportError(f"svl/_torch_ops.so is missing or does not match this torch: build it with semantic-ai_b200/build.py ({e})") from e


def _address(name: str) -> int:
    return ctypes.cast(getattr(_lib.lib(), name), ctypes.c_void_p).value


ops.bind(_address("svl_add_norm_f8_device"), _address("svl_f8_linear_device"), _address("svl_logits_rules_device"),
         _address("svl_last_error"), _lib.SvlError)


def of(stream, device):
    """`stream`, refused if it is not one of the tensors' device."""
    if stream.device != device:
        raise ValueError(f"stream must be one of {device}: got one of {stream.device}")
    return stream


def on(stream, device):
    """The context in which a call runs and allocates on `stream`, a stream of the tensors' device.
    (Outputs that belonged to another stream could be given out again while `stream` still writes.)"""
    return torch.cuda.stream(of(stream, device))
