"""The rules of a state's streams, changed between steps."""
import dataclasses
import time

import numpy as np
import pytest

from svl import LanguageModel, codec, config, synth
from svl._lib import SvlError
from svl.stt_pipeline import SttPipeline
from test_gpu_f8_model import check_rules

pytestmark = pytest.mark.gpu


def toy(wdt="f8", kv="bf16", layers=None, **kw):
    stt = config.stt_toy(**kw)
    cfg = stt.transformer(wdt, kv)
    if layers:
        cfg = dataclasses.replace(cfg, num_layers=layers)
    return stt, LanguageModel(stt, cfg, synth.stt_weights(stt, cfg, std=0.05))


@pytest.mark.parametrize("wdt", ["f8", "q8_0"])
@pytest.mark.parametrize("streams", [1, 5])
def test_rules_change_before_each_step(svl_lib, wdt, streams):
    """New penalties, biases and grammars of one stream or all take effect with the next step, with the same
    first_penalised as before and with another one."""
    stt, gm = toy(wdt, "f32")
    g = np.random.default_rng(7)
    plan = {}
    for i in range(1, 14):
        kw = dict(stream=int(g.integers(-1, streams)), first_penalised=int(i > 8), repetition=1 + float(g.integers(0, 4)) / 4,
                  frequency=float(g.integers(0, 3)) / 8, bias={int(v): float(g.integers(-4, 5)) / 2 for v in g.choice(stt.text_card, int(g.integers(0, 9)), replace=False)})
        if i % 3:
            kw["allowed"] = [int(v) for v in g.choice(stt.text_card, 20, replace=False)]
        plan[i] = [kw]
    check_rules(stt, gm, streams, 15, plan)


def test_rules_keep_the_captured_step(svl_lib):
    """A step is captured again only where the rules first come or first_penalised changes: an update of the others
    costs a fraction of a capture."""
    stt, gm = toy(layers=40)
    st = gm.init_state(1)
    audio = synth.audio_tokens(stt, 1)

    def median(rules):
        took = []
        for i in range(24):
            t = time.perf_counter()
            if rules:
                st.set_rules(**rules(i))
            gm.step([5], audio[0][None], st)
            took.append(time.perf_counter() - t)
        return np.median(took[4:])

    st.set_rules(repetition=1.5)
    step = median(None)
    kept = median(lambda i: dict(allowed=[5, 6, 7 + i], repetition=1.5 + i))
    captured = median(lambda i: dict(first_penalised=4 + i % 2))
    print(f"step {step * 1e6:.0f} us, with new rules {kept * 1e6:.0f}, captured again {captured * 1e6:.0f}")
    assert kept - step < 0.4 * (captured - step)


def test_pipeline_with_no_token_left(svl_lib):
    """A grammar that allows nothing: -1 for its stream, told by check() after the step that was fed it, and by no
    other; the other stream's tokens are those of a pipeline without rules."""
    import torch
    stt = config.stt_toy(card=2048, n_q=32)
    mcfg = codec.stt_mimi(codec.ENCODER)
    w = synth.mimi_weights(mcfg)
    w.update(synth.rvq_weights(32, 2048))
    cfg = stt.transformer("f32", "f32")
    mimi, q, lm = codec.Mimi(mcfg, w), codec.Quantizer(32, 2048, w), LanguageModel(stt, cfg, synth.stt_weights(stt, cfg))
    plain, ruled = SttPipeline(mimi, q, lm, 2), SttPipeline(mimi, q, lm, 2)
    ruled.lm_state.set_rules(stream=0, allowed=[])
    pcm = torch.from_numpy((0.3 * np.random.default_rng(1).standard_normal((4, 2, 1, mimi.frame_size))).astype(np.float32)).cuda()
    tokens = []
    for f in range(4):
        want, got = plain.step(pcm[f])[0], ruled.step(pcm[f])[0]
        torch.cuda.synchronize()
        tokens.append(got[0].item())
        assert got[1] == want[1]
        if f == 0:
            ruled.check()
        elif f == 1:
            with pytest.raises(SvlError, match="token"):
                ruled.check()
            ruled.check()
            ruled.lm_state.clear_rules(0)
    # Step 2 was still fed the -1 of step 1.
    assert tokens[:2] == [-1, -1] and tokens[2] >= 0 and tokens[3] >= 0
    with pytest.raises(SvlError, match="token"):
        ruled.check()
    plain.check()


def test_run_frames_with_no_token_left(svl_lib):
    """run_frames raises after its last frame; lm.step goes on with another token for that stream."""
    stt, gm = toy()
    st = gm.init_state(2)
    st.set_rules(stream=1, allowed=[])
    audio = synth.audio_tokens(stt, 4, streams=2)
    with pytest.raises(SvlError, match="token"):
        gm.run_frames(audio, st)
    assert [st.position(b) for b in range(2)] == [4, 4]
    with pytest.raises(SvlError, match="token"):
        gm.step([1, 0xFFFFFFFF], audio[0], st)
    assert st.position(0) == 4
    st.clear_rules(1)
    assert all(t < stt.text_card for t in gm.step([1, 2], audio[0], st))


def test_two_states_step_at_once(svl_lib):
    """Two e4m3 states of one model on two streams, one of them ruled, against each alone."""
    import ctypes

    import torch

    from svl import _lib
    stt, gm = toy(layers=6)
    audio = torch.from_numpy(synth.audio_tokens(stt, 30, streams=40).astype(np.int32)).cuda()
    text = torch.randint(0, stt.text_card, (30, 40), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(3))

    def run(together):
        states = [gm.init_state(40), gm.init_state(40)]
        states[1].set_rules(repetition=1.5, presence=1.0, first_penalised=0, bias={3: 0.5})
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        out = torch.empty(2, 30, 40, dtype=torch.int32, device="cuda")
        logits = torch.empty(2, 30, 40, stt.text_card, device="cuda")
        torch.cuda.synchronize()
        order = [(s, i) for i in range(30) for s in (0, 1)] if together else [(s, i) for s in (0, 1) for i in range(30)]
        for s, i in order:
            _lib.check(_lib.lib().svl_stt_step_device(gm.handle, states[s].handle, 40, *(ctypes.c_void_p(t.data_ptr()) for t in (text[i], audio[i], out[s, i], logits[s, i])),
                                                      ctypes.c_void_p(streams[s].cuda_stream)))
            if not together:
                streams[s].synchronize()
        for s in states:
            s.check()
        return out, logits

    alone, together = run(False), run(True)
    assert torch.equal(alone[0], together[0]) and torch.equal(alone[1], together[1])


def test_profiling_calls_take_an_e4m3_model(svl_lib):
    """svl_profile_kernels and svl_step_kernel_count of a ruled e4m3 state; after a reset it steps as before."""
    import ctypes

    from svl import _lib
    stt, gm = toy()
    st = gm.init_state(20)
    audio = synth.audio_tokens(stt, 3, streams=20)
    want = gm.run_frames(audio, st)
    for which in (0, 1):
        n = ctypes.c_int64()
        _lib.check(_lib.lib().svl_profile_kernels(gm.handle, st.handle, 20, which, 3, None, ctypes.byref(n)))
        assert n.value > 0
    st.check()
    counts = []
    for rules in (False, True):
        if rules:
            st.set_rules(repetition=2.0)
        k = ctypes.c_int32()
        _lib.check(_lib.lib().svl_step_kernel_count(gm.handle, st.handle, 20, ctypes.byref(k)))
        counts.append(k.value)
    assert counts[0] == counts[1] > 20  # the rules' kernel picks the token in either
    st.clear_rules()
    st.reset()
    np.testing.assert_array_equal(gm.run_frames(audio, st), want)
