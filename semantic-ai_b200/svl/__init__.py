"""semantic-voice-local's streaming LM step on B200 (sm_100a), through the C ABI.

The compute path is libsvl_b200.so (CUDA kernels + C++ host); this package is a thin
Python mirror of the reference's model API for tests, benchmarks and Python callers.
"""
from .config import (SttConfig, TransformerConfig, TtsConfig, pocket_tts, stt_1b, stt_2b6,
                     stt_toy)
from .model import FlowLm, LanguageModel, State

__all__ = ["SttConfig", "TransformerConfig", "TtsConfig", "LanguageModel", "FlowLm", "State",
           "stt_1b", "stt_2b6", "stt_toy", "pocket_tts", "add_norm_f8", "F8Linear", "logits_rules"]

# The operators on torch tensors import torch; the rest of the package does not need it.
_OPERATORS = {"add_norm_f8": "f8", "F8Linear": "f8", "logits_rules": "rules"}


def __getattr__(name):
    if name not in _OPERATORS:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    import importlib
    value = getattr(importlib.import_module("." + _OPERATORS[name], __name__), name)
    globals()[name] = value
    return value
