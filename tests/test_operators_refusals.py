"""What the 8-bit operators and the logits rules refuse, through the C ABI, without a GPU: every
check comes before any CUDA call, so bad arguments are told apart from a missing device."""
import ctypes

import pytest

from conftest import gpu_available

INVALID, CONFIG, CUDA, UNSUPPORTED = 2, 1, 3, 6
PTR = 4096  # a 16-byte aligned address that no refused call reads


def norm(lib, **change):
    a = dict(device=0, rows=4, k=256, dtype=0, x=PTR, xs=256, res=None, rs=0, norm=1, w=None, b=None, eps=1e-8, sum=None, ss=0,
             q=PTR, qs=256, scales=PTR, scs=4, stream=None)
    a.update(change)
    return lib.svl_add_norm_f8_device(*a.values())


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), INVALID), (dict(k=0), INVALID), (dict(k=32769, xs=32769, qs=32784), UNSUPPORTED), (dict(dtype=2), INVALID),
    (dict(dtype=-1), INVALID), (dict(norm=2), INVALID), (dict(norm=-2), INVALID), (dict(x=None), INVALID), (dict(q=None), INVALID),
    (dict(scales=None), INVALID), (dict(xs=255), INVALID), (dict(res=PTR, rs=255), INVALID), (dict(sum=PTR, ss=10), INVALID),
    (dict(qs=255), INVALID), (dict(qs=264), INVALID), (dict(q=PTR + 8), INVALID), (dict(scs=3), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID)])
def test_norm_refuses(svl_lib, change, status):
    assert norm(svl_lib, **change) == status
    assert svl_lib.svl_last_error()


def test_no_rows_is_no_work(svl_lib):
    assert norm(svl_lib, rows=0, x=None, q=None, scales=None) == 0
    assert svl_lib.svl_logits_rules_device(0, 0, 100, 0, None, 100, None, None, 0, None, None) == 0


def test_linear_refuses(svl_lib):
    from svl.config import CTensorView
    h = ctypes.c_void_p()
    data = (ctypes.c_float * 12)()
    views = (CTensorView * 2)(CTensorView(b"weight", ctypes.addressof(data), 12), CTensorView(b"bias", ctypes.addressof(data), 3))
    make = lambda n, k, count=2, out=ctypes.byref(h): svl_lib.svl_f8_linear_create(n, k, views, count, 0, out)  # noqa: E731
    assert make(3, 4, out=None) == INVALID
    assert make(0, 4) == CONFIG and make(3, 0) == CONFIG
    assert make(3, 5) == CONFIG              # 15 elements wanted
    assert make(4, 3) == CONFIG              # the bias has 3 elements, not 4
    assert make(3, 4, count=0) == CONFIG     # no weight
    assert make((1 << 24) + 1, 1) == UNSUPPORTED
    dev = lambda **c: svl_lib.svl_f8_linear_create_device(*dict(  # noqa: E731
        dict(n=128, k=128, w=PTR, ws=128, s=PTR, b=None, device=0, stream=None, out=ctypes.byref(h)), **c).values())
    assert dev(w=None) == INVALID and dev(s=None) == INVALID and dev(ws=127) == INVALID and dev(n=-1) == CONFIG
    assert not h.value
    assert svl_lib.svl_f8_linear_device(None, 1, PTR, 16, PTR, 1, 0, PTR, 1, None) == INVALID
    assert svl_lib.svl_f8_linear_error(None) == INVALID
    svl_lib.svl_f8_linear_destroy(None)


def rules(lib, rows=4, vocab=100, dtype=0, logits=PTR, stride=100, out=PTR, ostride=100, tokens=PTR, **fields):
    from svl.rules import CLogitsRules
    r = CLogitsRules(**fields)
    return lib.svl_logits_rules_device(0, rows, vocab, dtype, logits, stride, ctypes.byref(r), out, ostride, tokens, None)


@pytest.mark.parametrize("change", [
    dict(rows=-1), dict(vocab=0), dict(dtype=2), dict(logits=None), dict(out=None, tokens=None), dict(stride=99), dict(ostride=99),
    dict(d_history=PTR), dict(d_lengths=PTR), dict(append=1),
    dict(d_history=PTR, d_lengths=PTR, history_cap=0, history_stride=8),
    dict(d_history=PTR, d_lengths=PTR, history_cap=65536, history_stride=65536),
    dict(d_history=PTR, d_lengths=PTR, history_cap=8, history_stride=7),
    dict(d_bias_ids=PTR), dict(d_bias_values=PTR), dict(d_bias_ids=PTR, d_bias_values=PTR, bias_cap=65536, bias_stride=65536),
    dict(d_bias_ids=PTR, d_bias_values=PTR, bias_cap=-1), dict(d_bias_ids=PTR, d_bias_values=PTR, bias_cap=4, bias_stride=3),
    dict(d_masks=PTR, n_masks=4, mask_stride=3), dict(d_masks=PTR, n_masks=3, mask_stride=4), dict(d_masks=PTR, n_masks=-1, mask_stride=4)])
def test_rules_refuse(svl_lib, change):
    assert rules(svl_lib, **change) == INVALID
    assert svl_lib.svl_last_error()


@pytest.mark.skipif(gpu_available(), reason="checks the no-GPU failure path")
def test_good_calls_need_a_gpu(svl_lib):
    assert norm(svl_lib) == CUDA
    assert rules(svl_lib) == CUDA
    from svl.config import CTensorView
    data, h = (ctypes.c_float * 12)(), ctypes.c_void_p()
    assert svl_lib.svl_f8_linear_create(3, 4, (CTensorView * 1)(CTensorView(b"weight", ctypes.addressof(data), 12)), 1, 0,
                                        ctypes.byref(h)) == CUDA
    assert not h.value


def test_python_checks_come_first():
    """The torch entry points refuse tensors of the wrong place, type or shape by name."""
    import torch

    import svl
    cpu = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        svl.add_norm_f8(cpu)
    with pytest.raises(ValueError, match="weight must be a CUDA tensor"):
        svl.F8Linear(cpu, cpu)
    with pytest.raises(ValueError, match="logits must be a CUDA tensor"):
        svl.logits_rules(cpu)


def test_state_rules_refuse_without_a_state(svl_lib):
    from svl import _lib
    with pytest.raises(_lib.SvlError, match="null state"):
        _lib.check(svl_lib.svl_state_set_rules(None, -1, None))


@pytest.mark.parametrize("change", [dict(x=PTR + 2), dict(dtype=1, x=PTR + 1), dict(res=PTR + 2, rs=256), dict(sum=PTR + 1, ss=256),
                                    dict(w=PTR + 2), dict(b=PTR + 1), dict(scales=PTR + 2)])
def test_norm_refuses_misaligned(svl_lib, change):
    assert norm(svl_lib, **change) == INVALID
    assert b"aligned" in svl_lib.svl_last_error()


@pytest.mark.parametrize("change", [
    dict(logits=PTR + 2), dict(dtype=1, logits=PTR + 1), dict(out=PTR + 2), dict(tokens=PTR + 2), dict(d_dense_bias=PTR + 1),
    dict(d_history=PTR + 2, d_lengths=PTR, history_cap=8, history_stride=8), dict(d_history=PTR, d_lengths=PTR + 2, history_cap=8, history_stride=8),
    dict(d_bias_ids=PTR + 1, d_bias_values=PTR, bias_cap=4, bias_stride=4), dict(d_bias_ids=PTR, d_bias_values=PTR + 2, bias_cap=4, bias_stride=4),
    dict(d_masks=PTR + 2, n_masks=4, mask_stride=4), dict(d_mask_rows=PTR + 1), dict(d_repetition=PTR + 2)])
def test_rules_refuse_misaligned(svl_lib, change):
    assert rules(svl_lib, **change) == INVALID
    assert b"aligned" in svl_lib.svl_last_error()


def test_linear_create_refuses_misaligned(svl_lib):
    h = ctypes.c_void_p()
    for s, b in ((PTR + 2, None), (PTR, PTR + 1)):
        assert svl_lib.svl_f8_linear_create_device(128, 128, PTR, 128, s, b, 0, None, ctypes.byref(h)) == INVALID
        assert b"aligned" in svl_lib.svl_last_error()


@pytest.mark.parametrize("change,message", [(dict(b=PTR), b"bias"), (dict(norm=-1, b=PTR), b"bias"), (dict(norm=-1, w=PTR), b"weight"),
                                            (dict(norm=-1, w=PTR, b=PTR), b"weight")])
def test_norm_refuses_what_it_would_leave_out(svl_lib, change, message):
    """A weight without a norm, a bias of a norm that adds none."""
    assert norm(svl_lib, **change) == INVALID
    assert message in svl_lib.svl_last_error()
    assert norm(svl_lib, rows=0, **change) == 0


def test_linear_refuses_copies():
    """Two handles of one matrix would free it twice."""
    import copy
    import pickle

    import svl
    lin = svl.F8Linear.__new__(svl.F8Linear)  # no matrix: it is the copy that is refused
    for make in (copy.copy, copy.deepcopy, pickle.dumps, lambda x: copy.deepcopy({"head": x})):
        with pytest.raises(TypeError, match="cannot be copied"):
            make(lin)


@pytest.fixture
def set_rules(monkeypatch):
    """State.set_rules on a library that only records what it is given: the mask's allowed tokens."""
    import types

    import numpy as np

    from svl import _lib, model
    given = []

    def record(handle, stream, rules):
        r = ctypes.cast(rules, ctypes.POINTER(model.CSttRules)).contents
        words = np.array([r.allowed[i] for i in range(4)], np.uint32)
        given.append(np.flatnonzero(np.unpackbits(words.view(np.uint8), bitorder="little")).tolist())
        return 0

    monkeypatch.setattr(_lib, "lib", lambda: types.SimpleNamespace(svl_state_set_rules=record))
    state = model.State.__new__(model.State)
    state.handle, state.model = None, types.SimpleNamespace(stt=types.SimpleNamespace(text_card=100))
    return lambda allowed: (state.set_rules(allowed=allowed), given[-1])[1]


def test_allowed_tokens(set_rules):
    import numpy as np
    for allowed in ([5, 7, 99], (99, 5, 7), {5, 7, 99}, frozenset({5, 7, 99}), np.array([5, 7, 99], np.int16), [i in (5, 7, 99) for i in range(100)]):
        assert set_rules(allowed) == [5, 7, 99]
    assert set_rules([]) == set_rules(set()) == []
    assert set_rules(range(4, 40)) == list(range(4, 40))
    for wrong in ([1.5], [5.0, 7.0], [float("nan")], ["5"], [None], [-1], [100], [True] * 99):
        with pytest.raises(ValueError, match="allowed"):
            set_rules(wrong)
