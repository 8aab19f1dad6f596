"""The rules between logits and token on torch tensors: penalties for repeated tokens, biases,
grammar masks and the greedy pick (svl_logits_rules_device). For inference: logits that require a gradient are
taken, but the outputs are detached from them."""
from __future__ import annotations

import ctypes

from ._ops import on, ops


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
    token; mask_rows int32 [rows] chooses a row's mask (-1: none; without it, row r takes mask r).
    `out` must not overlap logits unless it is logits."""
    if stream is not None:
        with on(stream, logits.device):
            return logits_rules(logits, history, lengths, repetition, frequency, presence, dense_bias, bias_ids,
                                bias_values, masks, mask_rows, first_penalised, append, out)
    return ops.logits_rules(logits, history, lengths, repetition, frequency, presence, dense_bias, bias_ids, bias_values,
                            masks, mask_rows, first_penalised, append, out)
