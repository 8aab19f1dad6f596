"""STT models with e4m3 weights, and the rules behind the head of any STT model, on the GPU.

The 8-bit step is compared with a float64 restatement that rounds where the step rounds: weights to
e4m3 with a scale per block of 128 x 128, the input of every product to e4m3 with a scale per 128
columns, a bf16 ring's keys and values to bf16. Outside those roundings the step is f32, so both agree to about 1e-5 until a value lies
so near the middle between two e4m3 values that they round it apart: of about 2,000 rounded values
per step, whose spacing is 2^-3..2^-4 of them, some 2,000 * 1e-6 * 16 = 3 % of the steps hold one. From
there on the rings differ too, by the e4m3 rounding noise at most: 2^-4 / sqrt(3) = 3.6 % (rms) of an
operand at each of the products, which are 4 per layer and the head. So at most half the steps
of a run may be off by more than the quantised models' 2e-2 (||diff|| / ||reference||), none by
more than 3.6 % * sqrt(2 * 9 products) = 15 %.
"""
import dataclasses

import numpy as np
import pytest
import torch

from np_reference import Backbone
from svl import LanguageModel, config, synth
from svl._lib import SvlError
from test_gpu_rules import make as make_rules, reference as rules_reference

F = np.float32
gpu = pytest.mark.gpu


def e4m3(x):
    """f32 -> the nearest e4m3 value (ties to even), as f64."""
    return torch.from_numpy(np.ascontiguousarray(x, F)).to(torch.float8_e4m3fn).double().numpy()


def round_row(x):
    """A row as e4m3 with a scale per 128 columns."""
    x = x.astype(F)
    out = np.empty(len(x))
    for c in range(0, len(x), 128):
        top = max(F(np.abs(x[c:c + 128]).max()), F(2.0 ** -100))
        out[c:c + 128] = e4m3(x[c:c + 128] * (F(448) / top)) * float(top / F(448))
    return out


def round_matrix(w):
    w = w.astype(F)
    out = np.empty(w.shape)
    for r in range(0, w.shape[0], 128):
        for c in range(0, w.shape[1], 128):
            b = w[r:r + 128, c:c + 128]
            top = max(F(np.abs(b).max()), F(2.0 ** -100))
            out[r:r + 128, c:c + 128] = e4m3(b * (F(448) / top)) * float(top / F(448))
    return out


class Rounded:
    """W @ x with x rounded to an e4m3 row."""

    def __init__(self, w):
        self.w = round_matrix(w)

    def __matmul__(self, x):
        return self.w @ round_row(x)


class Bf16Ring(list):
    """A stream's keys or values, rounded to bf16 as they are stored."""

    def append(self, rows):
        super().append(torch.from_numpy(rows).float().bfloat16().double().numpy())


def logits_of(stt, cfg, w, text, audio):
    """Teacher-forced logits [steps, text_card] of one stream."""
    bb = Backbone(cfg, w)
    for name in list(bb.w):
        if any(s in name for s in ("in_proj", "out_proj", "linear_in", "linear_out", "linear1", "linear2")):
            bb.w[name] = Rounded(w[name])
    head = Rounded(w["text_linear.weight"])
    if cfg.kv_dtype == "bf16":
        bb.k, bb.v = [[Bf16Ring() for _ in range(cfg.num_layers)] for _ in "kv"]
    out = []
    for tt, au in zip(text, audio):
        x = w["text_emb.weight"][tt].astype(np.float64)
        for c in range(stt.n_q):
            x = x + w[f"emb.{c}.weight"][au[c]]
        x = bb.forward_token(x)
        out.append(head @ (x / np.sqrt((x * x).mean() + 1e-8) * w["out_norm.alpha"].reshape(-1)))
    return np.array(out)


def models():
    toy = config.stt_toy()
    odd = config.stt_toy(dim=320, num_heads=5, text_card=333, hidden_scale=3.3)  # hidden 704
    yield toy, toy.transformer("f8")
    yield odd, dataclasses.replace(odd.transformer("f8"), num_kv_heads=1)
    yield toy, dataclasses.replace(toy.transformer("f8"), norm_kind=config.NORM_LAYER, norm_eps=1e-5,
                                                      ffn_kind=config.FFN_PLAIN_GELU_TANH, ffn_hidden=300, context=None)
    yield toy, dataclasses.replace(toy.transformer("f8"), ffn_kind=config.FFN_PLAIN_GELU_ERF, ffn_hidden=200)


def close(got, want):
    rel = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)
    print(f"relative difference: median {np.median(rel):.2e}, largest {rel.max():.2e}")
    assert np.median(rel) <= 2e-2 and rel.max() <= 0.15


@gpu
@pytest.mark.parametrize("which", range(4))
def test_step(svl_lib, which):
    stt, cfg = list(models())[which]
    w = synth.stt_weights(stt, cfg, std=0.05)
    gm = LanguageModel(stt, cfg, w)
    st = gm.init_state(1, max_positions=64)
    steps = 30  # window 12: the ring wraps
    audio = synth.audio_tokens(stt, steps)
    text = np.random.default_rng(2).integers(0, stt.text_card, steps)
    got = []
    for i in range(steps):
        tok, lg = gm.step([text[i]], audio[i][None], st, logits=True)
        assert tok[0] == np.argmax(lg[0])
        got.append(lg[0])
    close(np.array(got), logits_of(stt, cfg, w, text, audio))


@gpu
@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("streams", [3, 20, 200])
def test_streams(svl_lib, streams, kv):
    """Every stream of a batch against the restatement."""
    stt = config.stt_toy()
    cfg = stt.transformer("f8", kv)
    w = synth.stt_weights(stt, cfg, std=0.05)
    gm = LanguageModel(stt, cfg, w)
    st = gm.init_state(streams)
    steps = 4
    audio = synth.audio_tokens(stt, steps, streams=streams)
    text = np.random.default_rng(3).integers(0, stt.text_card, (steps, streams))
    got = np.stack([gm.step(text[i], audio[i], st, logits=True)[1] for i in range(steps)])
    want = np.stack([logits_of(stt, cfg, w, text[:, b], audio[:, b]) for b in range(streams)], 1)
    close(got, want)


@gpu
def test_entry_points_agree(svl_lib):
    """run_frames and a loop of steps give the same tokens, twice; forward() is the step's layers."""
    stt = config.stt_toy(extra_heads_num_heads=2, extra_heads_dim=6)
    cfg = stt.transformer("f8")
    w = synth.stt_weights(stt, cfg, std=0.05)
    gm = LanguageModel(stt, cfg, w)
    audio = synth.audio_tokens(stt, 20, streams=5)
    runs = [gm.run_frames(audio, gm.init_state(5), extra=True) for _ in range(2)]
    np.testing.assert_array_equal(runs[0][0], runs[1][0])
    st = gm.init_state(5)
    prev = np.full(5, stt.text_card)
    for i in range(20):
        a = np.full((5, stt.n_q), stt.card, np.uint32) if i == 0 else audio[i]
        prev, ex = gm.step(prev, a, st, extra=True)
        np.testing.assert_array_equal(prev, runs[0][0][i])
        np.testing.assert_array_equal(ex, runs[0][1][i])
    x = np.random.default_rng(4).standard_normal((6, cfg.d_model)).astype(F)
    bb = Backbone(cfg, w)
    for name in list(bb.w):
        if any(s in name for s in ("in_proj", "out_proj", "linear_in", "linear_out")):
            bb.w[name] = Rounded(w[name])
    st2 = gm.init_state(2)
    close(gm.forward(x, st2, stream=1), np.array([bb.forward_token(r) for r in x]))


@gpu
def test_f8_model_refusals(svl_lib):
    stt = config.stt_toy()
    cfg = stt.transformer("f8")
    w = synth.stt_weights(stt, cfg)
    gm = LanguageModel(stt, cfg, w)
    with pytest.raises(SvlError, match="reference order"):
        gm.init_state(1, reference_order=True)
    scaled = dataclasses.replace(cfg, layer_scale=True)
    with pytest.raises(SvlError, match="layer scale"):
        LanguageModel(stt, scaled, synth.stt_weights(stt, scaled))
    st = gm.init_state(2)
    for kw, what in [(dict(repetition=0.0), "repetition"), (dict(repetition=float("nan")), "penalties"),
                     (dict(frequency=float("inf")), "penalties"), (dict(first_penalised=-1), "first_penalised"),
                     (dict(bias={stt.text_card: 1.0}), "biased token"), (dict(bias={i: 1.0 for i in range(257)}), "n_bias"),
                     (dict(stream=2), "stream")]:
        with pytest.raises(SvlError, match=what):
            st.set_rules(**kw)
    with pytest.raises(ValueError):
        st.set_rules(allowed=np.ones(3, bool))
    with pytest.raises(ValueError):
        st.set_rules(allowed=[stt.text_card])


def check_rules(stt, gm, streams, steps, plan, st=None):
    """Steps two states on the same inputs, one with rules: `plan` maps a step to the keyword
    arguments of set_rules calls before it. The ruled logits must be the rules applied to the
    other state's logits, value for value."""
    V = stt.text_card
    plain, ruled = gm.init_state(streams), st or gm.init_state(streams)
    audio = synth.audio_tokens(stt, steps, streams=streams)
    text = np.random.default_rng(6).integers(0, V, (steps, streams))
    r = {"history": np.full((streams, 1024), -1, np.int32), "lengths": np.zeros(streams, np.int32),
         "repetition": np.ones(streams, F), "frequency": np.zeros(streams, F), "presence": np.zeros(streams, F),
         "bias_ids": np.full((streams, 256), -1, np.int32), "bias_values": np.zeros((streams, 256), F),
         "masks": np.full((streams, (V + 31) // 32), -1, np.int32), "mask_rows": np.full(streams, -1, np.int32), "append": True}
    on = False
    for i in range(steps):
        for kw in plan.get(i, []):
            ruled.set_rules(**kw)
            on = True
            r["first_penalised"] = kw.get("first_penalised", 4)
            for b in range(streams) if kw.get("stream", -1) < 0 else [kw["stream"]]:
                r["repetition"][b], r["frequency"][b] = kw.get("repetition", 1), kw.get("frequency", 0)
                r["presence"][b] = kw.get("presence", 0)
                r["bias_ids"][b], r["bias_values"][b] = -1, 0
                for j, (k, v) in enumerate(kw.get("bias", {}).items()):
                    r["bias_ids"][b, j], r["bias_values"][b, j] = k, v
                r["mask_rows"][b] = -1
                if "allowed" in kw:
                    ok = np.zeros(r["masks"].shape[1] * 32, np.uint8)
                    ok[list(kw["allowed"])] = 1
                    r["masks"][b], r["mask_rows"][b] = np.packbits(ok, bitorder="little").view(np.int32), b
        _, lg = gm.step(text[i], audio[i], plain, logits=True)
        tok, got = gm.step(text[i], audio[i], ruled, logits=True)
        if not on:
            np.testing.assert_array_equal(got, lg)
            continue
        want, tokens, r["history"], r["lengths"] = rules_reference(lg, r)
        np.testing.assert_array_equal(got, want, err_msg=f"step {i}")
        np.testing.assert_array_equal(tok.view(np.int32), tokens)
    return ruled, r


@gpu
@pytest.mark.parametrize("wdt,kv", [("f32", "f32"), ("q8_0", "f32"), ("bf16", "bf16"), ("f8", "bf16")])
@pytest.mark.parametrize("streams", [1, 3, 80])
def test_rules_in_the_step(svl_lib, wdt, kv, streams):
    stt = config.stt_toy(extra_heads_num_heads=1, extra_heads_dim=4)
    cfg = stt.transformer(wdt, kv)
    gm = LanguageModel(stt, cfg, synth.stt_weights(stt, cfg, std=0.05))
    plan = {1: [dict(repetition=1.5, frequency=0.25, presence=0.5, first_penalised=0)],
            4: [dict(stream=streams - 1, repetition=1.25, bias={7: 3.5, 99: -2.0}, first_penalised=0)],
            6: [dict(stream=0, allowed=[3, 50, 98], presence=2.0, first_penalised=3)],
            9: [dict(stream=0, allowed=[], first_penalised=3)]}
    check_rules(stt, gm, streams, 12, plan)


@gpu
def test_rules_reset_copy_clear(svl_lib):
    stt = config.stt_toy()
    cfg = stt.transformer("f8")
    gm = LanguageModel(stt, cfg, synth.stt_weights(stt, cfg, std=0.05))
    kw = dict(repetition=2.0, presence=1.0, first_penalised=0)
    a, _ = check_rules(stt, gm, 3, 8, {0: [kw]})
    audio = synth.audio_tokens(stt, 2, seed=9)
    step = lambda s, n: gm.step(np.full(n, 5), np.repeat(audio[1][None], n, 0), s, logits=True)
    # A copied stream goes on as its source does.
    b = gm.init_state(3)
    b.set_rules(**kw)
    b.copy_from(a, 2, 0)
    (_, la), (_, lb) = step(a, 3), step(b, 1)
    np.testing.assert_array_equal(la[2], lb[0])
    # Reset: nothing said, so a fresh state's logits.
    a.reset(1)
    fresh, plain = gm.init_state(3), gm.init_state(3)
    fresh.set_rules(**kw)
    np.testing.assert_array_equal(step(a, 2)[1][1], step(fresh, 2)[1][1])
    np.testing.assert_array_equal(step(plain, 1)[1][0], gm.step([5], audio[1][None], gm.init_state(1), logits=True)[1][0])
    # Cleared rules: an unruled state's logits.
    a.reset()
    a.clear_rules()
    plain.reset()
    np.testing.assert_array_equal(step(a, 3)[1], step(plain, 3)[1])


@gpu
def test_no_token_left(svl_lib):
    """No allowed token: 0xFFFFFFFF, which the next step refuses on the device, as any token out of range."""
    stt = config.stt_toy()
    cfg = stt.transformer("f8")
    gm = LanguageModel(stt, cfg, synth.stt_weights(stt, cfg))
    st = gm.init_state(1)
    st.set_rules(allowed=[])
    audio = synth.audio_tokens(stt, 3, streams=1)
    assert gm.step([0], audio[0], st)[0] == 0xFFFFFFFF
    with pytest.raises(SvlError):
        gm.step([0xFFFFFFFF], audio[0], st)
    with pytest.raises(SvlError):
        gm.run_frames(audio, st)


@gpu
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_norm_linear_rules_together(svl_lib, rows):
    """A head as its user writes it: norm to e4m3, product, rules; in one captured graph too."""
    import svl
    g = np.random.default_rng(rows)
    d, vocab = 640, 1500
    w = round_matrix(g.standard_normal((vocab, d)).astype(F) * 0.05)
    top = np.array([[np.abs(w[r:r + 128, c:c + 128]).max() for c in range(0, d, 128)] for r in range(0, vocab, 128)])
    scales = torch.from_numpy((top / 448).astype(F))
    full = np.repeat(np.repeat(scales.numpy(), 128, 0)[:vocab], 128, 1)[:, :d]
    wq = torch.from_numpy((w / full).astype(F)).to(torch.float8_e4m3fn)
    w = wq.double().numpy() * full
    x, res = g.standard_normal((2, rows, d)).astype(F)
    alpha = (1 + 0.1 * g.standard_normal(d)).astype(F)
    dev = lambda a: torch.from_numpy(a).cuda()
    lin = svl.F8Linear(wq.cuda(), scales.cuda())
    _, r = make_rules(rows, vocab, 3, history=40, biased=9, masks=2)
    rd = {k: dev(v.copy()) if isinstance(v, np.ndarray) else v for k, v in r.items()}
    xd, resd, ad = dev(x), dev(res), dev(alpha)

    def head():
        q, s, h = svl.add_norm_f8(xd, resd, "rms", ad, eps=1e-8)
        lg = lin(q, s, out_dtype=torch.float32)
        return h, lg, *svl.logits_rules(lg, **rd)

    h, lg, out, tok = [t.cpu().numpy() for t in head()]
    np.testing.assert_array_equal(h, x + res)
    z = (x + res).astype(np.float64)
    z = z / np.sqrt((z * z).mean(1, keepdims=True) + 1e-8) * alpha
    close(lg, np.stack([w @ round_row(v) for v in z]))
    want, tokens, _, _ = rules_reference(lg, r)
    np.testing.assert_array_equal(out, want)
    np.testing.assert_array_equal(tok, tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = head()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip((h, lg, out, tok), again):
        np.testing.assert_array_equal(a, b.cpu().numpy())


@gpu
def test_rules_in_reference_order(svl_lib):
    """The rules read the logits that a state in reference order gives."""
    stt = config.stt_toy()
    cfg = stt.transformer("q8_0")
    gm = LanguageModel(stt, cfg, synth.stt_weights(stt, cfg, std=0.05))
    a, b = (gm.init_state(1, reference_order=True) for _ in range(2))
    b.set_rules(allowed=[5, 6], bias={6: 100.0})
    audio = synth.audio_tokens(stt, 1)
    _, la = gm.step([1], audio, a, logits=True)
    tok, lb = gm.step([1], audio, b, logits=True)
    assert tok[0] == 6 and lb[0, 5] == la[0, 5] and lb[0, 6] == F(la[0, 6] + F(100))
    assert np.all(np.isneginf(np.delete(lb[0], [5, 6])))


@gpu
def test_first_calls_captured(svl_lib):
    """A process whose very first calls are made while a graph is captured."""
    import subprocess
    import sys
    code = """
import torch, svl
from svl import _lib
lib = _lib.lib()
w = torch.eye(256, device="cuda").to(torch.float8_e4m3fn)
lin = svl.F8Linear(w, torch.ones(2, 2, device="cuda"))
shapes = ((1, 256), (40, 256), (200, 256), (3000, 256))
xs = [torch.randn(s, device="cuda") for s in shapes]
big = [torch.randn(3, 131072, device="cuda"), torch.randn(300, 40000, device="cuda").bfloat16()]
hist = torch.zeros(3, 9000, dtype=torch.int32, device="cuda"), torch.full((3,), 9000, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    outs = [lin(*svl.add_norm_f8(x, x)[:2]) for x in xs]
    rules = [svl.logits_rules(big[0], history=hist[0], lengths=hist[1]), svl.logits_rules(big[1])]
g.replay()
torch.cuda.synchronize()
for x, o in zip(xs, outs):
    assert torch.equal(o, lin(*svl.add_norm_f8(x, x)[:2]))
assert torch.equal(rules[0][1], svl.logits_rules(big[0], history=hist[0], lengths=hist[1])[1])
assert torch.equal(rules[1][1].long(), big[1].float().argmax(1))
print("captured")
"""
    import os
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
