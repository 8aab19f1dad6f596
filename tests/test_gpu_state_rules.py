"""The rules of a state's streams, changed between steps."""
import dataclasses
import time

import numpy as np
import pytest

from svl import LanguageModel, config, synth
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
