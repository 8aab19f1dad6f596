"""The 8-bit step against its float64 restatement, tightly enough to tell it from a step with one thing wrong.

Outside its roundings to e4m3 and bf16 the step is f32: a chain of some 30 operations over up to 704 terms, whose
roundings of 2^-24 each add up at random to well below 1e-5 of a row. A value that lies within that of the middle
between two e4m3 values is rounded apart: of about 2,000 rounded values per step some 2,000 * 1e-6 * 16 = 3 %
of the steps hold one, and a stream keeps it in its ring. After n steps at most 3 n % of the streams are affected: over
three steps 6 % on average. So at least 80 % of the (step, stream) pairs must agree to 1e-5, and a restatement with one
mistake must not: a mistake moves every row.
"""
import dataclasses

import numpy as np
import pytest
import torch

from np_reference import Backbone
from svl import LanguageModel, config, synth
from test_gpu_f8_model import Bf16Ring, round_matrix, round_row

pytestmark = pytest.mark.gpu

F = np.float32
STREAMS, STEPS = 60, 3


class Product:
    """W @ x of an e4m3 matrix; x rounded by `rows`."""

    def __init__(self, w, rows):
        self.w, self.rows = w, rows

    def __matmul__(self, x):
        return self.w @ self.rows(x)


def half_blocks(x):
    return np.concatenate([round_row(x[c:c + 64]) for c in range(0, len(x), 64)])


MISTAKES = {
    "none": {},
    "the other GELU": dict(gelu=True),
    "no eps": dict(eps=True),
    "no rounding of the ring": dict(ring=True),
    "in_proj's input not rounded": dict(rows={"in_proj": lambda x: x}),
    "out_proj's input not rounded": dict(rows={"out_proj": lambda x: x}),
    "linear_out's input not rounded": dict(rows={"linear_out": lambda x: x, "linear2": lambda x: x}),
    "the head's input not rounded": dict(rows={"text_linear": lambda x: x}),
    "a scale per 64 columns": dict(rows={"linear_in": half_blocks, "linear1": half_blocks}),
    "matrices not rounded": dict(matrices=True),
}


def restated(stt, cfg, w, rounded, text, audio, gelu=False, eps=False, ring=False, rows={}, matrices=False):
    """Teacher-forced logits [steps, text_card] of one stream; `rounded`: the e4m3 matrices by name."""
    if gelu:
        cfg = dataclasses.replace(cfg, ffn_kind={0: 1, 1: 0}[cfg.ffn_kind])
    if eps:
        cfg = dataclasses.replace(cfg, norm_eps=0.0)
    bb = Backbone(cfg, w)
    name_of = lambda name: next((s for s in ("in_proj", "out_proj", "linear_in", "linear_out", "linear1", "linear2", "text_linear") if s in name), "")  # noqa: E731
    product = lambda name: Product(w[name].astype(np.float64) if matrices else rounded[name], rows.get(name_of(name), round_row))  # noqa: E731
    for name in rounded:
        if name in bb.w and name != "text_linear.weight":
            bb.w[name] = product(name)
    head = product("text_linear.weight")
    if cfg.kv_dtype == "bf16" and not ring:
        bb.k, bb.v = [[Bf16Ring() for _ in range(cfg.num_layers)] for _ in "kv"]
    out = []
    for tt, au in zip(text, audio):
        x = w["text_emb.weight"][tt].astype(np.float64)
        for c in range(stt.n_q):
            x = x + w[f"emb.{c}.weight"][au[c]]
        x = bb.forward_token(x)
        out.append(head @ (x / np.sqrt((x * x).mean() + 1e-8) * w["out_norm.alpha"].reshape(-1)))
    return np.array(out)


def near(got, want):
    """The share of rows that agree to 1e-5 and the largest difference, relative."""
    rel = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)
    return (rel <= 1e-5).mean(), rel.max()


def models():
    toy = config.stt_toy()
    odd = config.stt_toy(dim=320, num_heads=5, text_card=333, hidden_scale=3.3)  # hidden 704
    some = ["none", "in_proj's input not rounded", "out_proj's input not rounded", "linear_out's input not rounded",
            "the head's input not rounded", "a scale per 64 columns", "matrices not rounded"]
    yield "silu, bf16 ring", odd, dataclasses.replace(odd.transformer("f8", "bf16"), num_kv_heads=1, norm_eps=1e-3), some + ["no rounding of the ring", "no eps"]
    yield "silu, f32 ring", toy, toy.transformer("f8"), some
    yield "tanh, layer norm", toy, dataclasses.replace(toy.transformer("f8"), norm_kind=config.NORM_LAYER, norm_eps=1e-3, ffn_kind=config.FFN_PLAIN_GELU_TANH,
                                                       ffn_hidden=300, context=None), some + ["the other GELU", "no eps"]
    yield "erf", toy, dataclasses.replace(toy.transformer("f8"), ffn_kind=config.FFN_PLAIN_GELU_ERF, ffn_hidden=200), ["none", "the other GELU"]


@pytest.mark.parametrize("which", range(4))
def test_the_step_and_no_other(svl_lib, which):
    name, stt, cfg, mistakes = list(models())[which]
    # Weights of a size at which the activations' curves show: pre-activations of order 1.
    w = synth.stt_weights(stt, cfg, std=0.1)
    rounded = {n: round_matrix(v) for n, v in w.items()
               if any(s in n for s in ("in_proj", "out_proj", "linear_in", "linear_out", "linear1", "linear2", "text_linear"))}
    gm = LanguageModel(stt, cfg, w)
    st = gm.init_state(STREAMS, max_positions=STEPS)
    audio = synth.audio_tokens(stt, STEPS, streams=STREAMS)
    text = np.random.default_rng(3).integers(0, stt.text_card, (STEPS, STREAMS))
    got = np.stack([gm.step(text[i], audio[i], st, logits=True)[1] for i in range(STEPS)])
    for mistake in mistakes:
        kw = MISTAKES[mistake]
        want = np.stack([restated(stt, cfg, w, rounded, text[:, b], audio[:, b], **kw) for b in range(STREAMS)], 1)
        share, worst = near(got, want)
        print(f"{name}, {mistake}: {share:.1%} within 1e-5, largest {worst:.1e}")
        if mistake == "none":
            assert share >= 0.8 and worst <= 0.15
        else:
            assert share < 0.8


@pytest.mark.parametrize("rows", [5, 300])
def test_norm_and_product(svl_lib, rows):
    """svl.add_norm_f8 and svl.F8Linear as a head: 640 rounded values per row, 1 % of the rows hold one that may be
    rounded apart. A restatement without eps or without the rows' rounding is told apart."""
    import svl
    g = np.random.default_rng(rows)
    d, n, eps = 640, 500, 1e-3
    w = round_matrix(g.standard_normal((n, d)).astype(F) * 0.05)
    x, res = g.standard_normal((2, rows, d)).astype(F)
    alpha = (1 + 0.1 * g.standard_normal(d)).astype(F)
    top = np.array([[np.abs(w[r:r + 128, c:c + 128]).max() for c in range(0, d, 128)] for r in range(0, n, 128)])
    scales = torch.from_numpy((top / 448).astype(F))
    full = np.repeat(np.repeat(scales.numpy(), 128, 0)[:n], 128, 1)[:, :d]
    wq = torch.from_numpy((w / full).astype(F)).to(torch.float8_e4m3fn)
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    q, s, h = svl.add_norm_f8(dev(x), dev(res), "rms", dev(alpha), eps=eps)
    got = svl.F8Linear(wq.cuda(), scales.cuda())(q, s).cpu().numpy()
    w64, h64 = wq.double().numpy() * full, (x + res).astype(np.float64)
    norm = lambda e: h64 / np.sqrt((h64 * h64).mean(1, keepdims=True) + e) * alpha  # noqa: E731
    share, worst = near(got, np.stack([w64 @ round_row(v) for v in norm(eps)]))
    print(f"{rows} rows: {share:.1%} within 1e-5, largest {worst:.1e}")
    assert share >= 0.8 and worst <= 0.15
    assert near(got, np.stack([w64 @ round_row(v) for v in norm(0.0)]))[0] < 0.8
    assert near(got, norm(eps) @ w64.T)[0] < 0.8
