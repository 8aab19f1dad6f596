"""The rules between logits and token on torch tensors: penalties for repeated tokens, biases,
grammar masks and the greedy pick (svl_logits_rules_device)."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .f8 import _DTYPES, _row_stride, _rows, _stream, _vector

_INTS = (torch.int32,)


class CLogitsRules(ctypes.Structure):
    """svl_logits_rules (include/svl_cuda.h)."""
    _fields_ = [("d_history", ctypes.c_void_p), ("history_stride", ctypes.c_int64), ("d_lengths", ctypes.c_void_p),
                ("history_cap", ctypes.c_int32), ("first_penalised", ctypes.c_int32),
                ("d_repetition", ctypes.c_void_p), ("d_frequency", ctypes.c_void_p), ("d_presence", ctypes.c_void_p),
                ("d_dense_bias", ctypes.c_void_p), ("d_bias_ids", ctypes.c_void_p), ("d_bias_values", ctypes.c_void_p),
                ("bias_stride", ctypes.c_int64), ("bias_cap", ctypes.c_int32), ("n_masks", ctypes.c_int32),
                ("d_masks", ctypes.c_void_p), ("mask_stride", ctypes.c_int64), ("d_mask_rows", ctypes.c_void_p),
                ("append", ctypes.c_int32), ("_pad", ctypes.c_int32)]


def logits_rules(logits, history=None, lengths=None, repetition=None, frequency=None, presence=None, dense_bias=None,
                 bias_ids=None, bias_values=None, masks=None, mask_rows=None, first_penalised: int = 0,
                 append: bool = False, out=None, stream=None):
    """Applies the rules that are given to logits (CUDA [rows, vocab], float32 or bfloat16) and
    picks each row's token. Returns (logits after the rules, tokens int32 [rows]; -1 where no
    token may follow). `out` takes the logits (it may be `logits`).

    history int32 [rows, cap], lengths int32 [rows]: each row's ring of past tokens and how many
    were ever recorded; repetition, frequency, presence float32 [rows]: the penalties of a token
    that occurs c > 0 times (l / repetition or l * repetition, then - (frequency * c + presence)).
    Ids below first_penalised are never penalised; append records the picked tokens.
    dense_bias float32 [vocab]; bias_ids int32 and bias_values float32 [rows, entries] (ids
    outside the vocabulary are pads). masks int32 [n, words of 32 tokens], a set bit allows its
    token; mask_rows int32 [rows] chooses a row's mask (-1: none; without it, row r takes mask r)."""
    _rows("logits", logits)
    rows, vocab = logits.shape
    device = logits.device
    r = CLogitsRules()
    if history is not None or lengths is not None:
        if history is None or lengths is None:
            raise ValueError("history and lengths go together")
        _rows("history", history, (rows, history.shape[1]), _INTS)
        _same(device, history=history)
    if history is not None and (history.shape[1] or append):
        r.d_history, r.history_stride, r.history_cap = history.data_ptr(), _row_stride(history), history.shape[1]
        r.d_lengths = _ints("lengths", lengths, rows, device)
    r.d_repetition = _vector("repetition", repetition, rows, device)
    r.d_frequency = _vector("frequency", frequency, rows, device)
    r.d_presence = _vector("presence", presence, rows, device)
    r.d_dense_bias = _vector("dense_bias", dense_bias, vocab, device)
    if bias_ids is not None or bias_values is not None:
        if bias_ids is None or bias_values is None:
            raise ValueError("bias_ids and bias_values go together")
        _rows("bias_ids", bias_ids, (rows, bias_ids.shape[1]), _INTS)
        _rows("bias_values", bias_values, bias_ids.shape, (torch.float32,))
        _same(device, bias_ids=bias_ids, bias_values=bias_values)
        if rows > 1 and bias_ids.stride(0) != bias_values.stride(0):
            raise ValueError("bias_ids and bias_values must have the same row stride")
        r.d_bias_ids, r.d_bias_values = bias_ids.data_ptr(), bias_values.data_ptr()
        r.bias_stride, r.bias_cap = _row_stride(bias_ids), bias_ids.shape[1]
    if masks is not None:
        _rows("masks", masks, (masks.shape[0], max(masks.shape[1], (vocab + 31) // 32)), _INTS)
        _same(device, masks=masks)
        r.d_masks, r.mask_stride, r.n_masks = masks.data_ptr(), _row_stride(masks), masks.shape[0]
    if mask_rows is not None:
        r.d_mask_rows = _ints("mask_rows", mask_rows, rows, device)
    r.first_penalised, r.append = first_penalised, int(append)
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=device)
    else:
        _rows("out", out, logits.shape, (logits.dtype,))
        _same(device, out=out)
    tokens = torch.empty((rows,), dtype=torch.int32, device=device)
    _lib.check(_lib.lib().svl_logits_rules_device(
        device.index, rows, vocab, _DTYPES[logits.dtype], logits.data_ptr(), _row_stride(logits), ctypes.byref(r),
        out.data_ptr(), _row_stride(out), tokens.data_ptr(), _stream(stream, device)))
    return out, tokens


def _same(device, **tensors):
    for name, t in tensors.items():
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, the logits on {device}")


def _ints(name: str, t, n: int, device):
    if t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be {n} contiguous int32 values on {device}: got {tuple(t.shape)}, {t.dtype}, {t.device}")
    return t.data_ptr()
