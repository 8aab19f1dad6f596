"""What the 8-bit decode step's operators cost: the norm that writes 8-bit rows, the product that
reads them, and the rules between the logits and the token.

Each operator has a plain form in elementary torch operations and the framework's own call. The
cases stand for a streaming speech model's step at 1 to 512 streams (widths 1024 to 2560,
feed-forward rows of 5632 to 20480, text vocabularies of 4000 and 8000), for prompts of up to
16384 rows, and for larger vocabularies.
"""
import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
BLOCK = 128         # columns (and weight rows) that share a scale
TINY = 2.0 ** -100  # the least largest value a group's scale is made from
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _svl():
    """The framework's package, from the tree this runs in."""
    path = os.path.join(os.getcwd(), "semantic-ai_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import svl
    return svl


def _blocks(n):
    return -(-n // BLOCK)


def listed():
    return [
        # One stream's step: the f32 residual stream of a width-2048 model, a chain of small launches.
        {"name": "norm 1x2048 f32", "op": "norm", "rows": 1, "k": 2048, "dtype": "f32", "norm": "rms", "residual": True},
        # 512 Pocket-TTS streams: LayerNorm of width 1024.
        {"name": "norm 512x1024 layer f32", "op": "norm", "rows": 512, "k": 1024, "dtype": "f32", "norm": "layer", "residual": True},
        # An attention output or hidden rows on their way into a product: no norm, odd sizes.
        {"name": "quantise 333x5637 bf16", "op": "norm", "rows": 333, "k": 5637, "dtype": "bf16", "norm": "none", "residual": False},
        # Long prompts of many streams at once.
        {"name": "norm 16384x2560 bf16", "op": "norm", "rows": 16384, "k": 2560, "dtype": "bf16", "norm": "rms", "residual": True},
        # One stream: the feed-forward input product, bound by its weights' bytes.
        {"name": "linear 1x11264x2048", "op": "linear", "rows": 1, "n": 11264, "k": 2048, "out": "f32", "bias": False},
        # A few streams on the narrow product that needs its long axis split.
        {"name": "linear 37x2048x5632", "op": "linear", "rows": 37, "n": 2048, "k": 5632, "out": "f32", "bias": False},
        # 256 streams: the fused query, key and value product.
        {"name": "linear 256x6144x2048", "op": "linear", "rows": 256, "n": 6144, "k": 2048, "out": "bf16", "bias": False},
        # Ragged in every size, with a bias: 4001 text rows.
        {"name": "linear 515x4001x2500", "op": "linear", "rows": 515, "n": 4001, "k": 2500, "out": "f32", "bias": True},
        # A long prompt through the feed-forward input: bound by the tensor cores.
        {"name": "linear 8192x11264x2048", "op": "linear", "rows": 8192, "n": 11264, "k": 2048, "out": "bf16", "bias": False},
        # One stream of the 8000-token model.
        {"name": "rules 1x8000 f32", "op": "rules", "rows": 1, "vocab": 8000, "dtype": "f32", "history": 250, "biased": 16, "dense": False, "masks": 1},
        # 256 streams of the 4001-token model, whose rows do not start on 16 bytes.
        {"name": "rules 256x4001 f32", "op": "rules", "rows": 256, "vocab": 4001, "dtype": "f32", "history": 750, "biased": 64, "dense": True, "masks": 8},
        # A large vocabulary, a long history, bf16 logits.
        {"name": "rules 192x131072 bf16", "op": "rules", "rows": 192, "vocab": 131072, "dtype": "bf16", "history": 2048, "biased": 128, "dense": True, "masks": 192},
    ]


def _log_int(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "rules"])
    if op == "norm":
        k = _log_int(rng, 64, 11264)
        return {"op": op, "rows": _log_int(rng, 1, min(16384, 16384 * 2560 // k)), "k": k, "dtype": rng.choice(["f32", "bf16"]),
                "norm": rng.choice(["rms", "rms", "layer", "none"]), "residual": rng.random() < 0.7}
    if op == "linear":
        n, k = _log_int(rng, 96, 20480), _log_int(rng, 64, 11264)
        return {"op": op, "rows": _log_int(rng, 1, min(8192, 8192 * 11264 * 2048 // (n * k))), "n": n, "k": k,
                "out": rng.choice(["f32", "bf16"]), "bias": rng.random() < 0.4}
    vocab = _log_int(rng, 1000, 131072)
    rows = _log_int(rng, 1, min(512, 192 * 131072 // vocab // 2))
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "bf16"]), "history": rng.choice([0, _log_int(rng, 1, 2048)]),
            "biased": rng.choice([0, rng.randint(1, 128)]), "dense": rng.random() < 0.5, "masks": rng.choice([0, 1, rng.randint(1, rows)])}


def _prepare_norm(case, make):
    rows, k, dtype = case["rows"], case["k"], DTYPES[case["dtype"]]
    # A residual stream: a few columns carry much larger values than the rest.
    x = make(rows, k) * (1.0 + 20.0 * (make(k).abs() > 2.5))
    state = {"x": x.to(dtype), "residual": (0.3 * make(rows, k)).to(dtype) if case["residual"] else None, "weight": None, "bias": None}
    if case["norm"] != "none":
        state["weight"] = 1.0 + 0.1 * make(k)
    if case["norm"] == "layer":
        state["bias"] = 0.1 * make(k)
    return state


def _prepare_linear(case, make):
    rows, n, k = case["rows"], case["n"], case["k"]
    kb, nb = _blocks(k), _blocks(n)
    pad = lambda t, r: torch.nn.functional.pad(t, (0, kb * BLOCK - k, 0, r - t.shape[0]))  # noqa: E731
    # The weights as a program holds them: e4m3 with a scale for each 128 x 128 block.
    w = pad(0.02 * make(n, k), nb * BLOCK).view(nb, BLOCK, kb, BLOCK)
    a = w.abs().amax((1, 3)).clamp_min(TINY)
    wq = (w * (448.0 / a)[:, None, :, None]).clamp(-448, 448).to(E4M3).view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous()
    # Activations as the norm before leaves them: e4m3 with a scale for each row and 128 columns.
    x = pad(make(rows, k), rows).view(rows, kb, BLOCK)
    b = x.abs().amax(2).clamp_min(TINY)
    store = torch.zeros(rows, -(-k // 16) * 16, device=x.device).to(E4M3)
    store[:, :k] = (x * (448.0 / b)[:, :, None]).clamp(-448, 448).to(E4M3).view(rows, kb * BLOCK)[:, :k]
    state = {"q": store[:, :k], "scales": (b / 448.0).t().contiguous(), "weight": wq, "weight_scales": a / 448.0,
             "bias": 0.1 * make(n) if case["bias"] else None, "out": DTYPES[case["out"]], "linear": None}
    if own:  # the handle a program makes once from its weights
        state["linear"] = _svl().F8Linear(wq, state["weight_scales"], state["bias"])
    return state


def _prepare_rules(case, make, gen):
    rows, vocab, cap, biased = case["rows"], case["vocab"], case["history"], case["biased"]
    dev = gen.device
    ints = lambda high, *shape: torch.randint(0, high, shape, generator=gen, device=dev)  # noqa: E731
    state = {"logits": (3.0 * make(rows, vocab)).to(DTYPES[case["dtype"]])}
    if cap:
        # What a stream has said: few words often, and some positions not used yet.
        rare = ints(vocab, rows, cap)
        state["history"] = torch.where(torch.rand(rows, cap, generator=gen, device=dev) < 0.5, rare % min(vocab, 40), rare).to(torch.int32)
        state["lengths"] = ints(2 * cap + 1, rows).to(torch.int32)  # over the ring's size: it has wrapped
        state["repetition"] = 1.0 + 0.5 * torch.rand(rows, generator=gen, device=dev)
        state["frequency"] = 0.2 * torch.rand(rows, generator=gen, device=dev)
        state["presence"] = 0.5 * torch.rand(rows, generator=gen, device=dev)
    if biased:
        step = vocab // biased
        ids = torch.arange(biased, device=dev) * step + ints(step, rows, biased)  # each id once
        state["bias_ids"] = ids.to(torch.int32)
        state["bias_values"] = 2.0 * make(rows, biased)
    if case["dense"]:
        state["dense_bias"] = 0.5 * make(vocab)
    if case["masks"]:
        words = -(-vocab // 32)
        bits = torch.rand(case["masks"], words * 32, generator=gen, device=dev) < 0.25
        weights = torch.ones(32, dtype=torch.int64, device=dev) << torch.arange(32, device=dev)
        packed = (bits.view(case["masks"], words, 32) * weights).sum(2)
        state["masks"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
        if rows > 8:
            state["masks"][-1] = 0  # a grammar with no way on
        state["mask_rows"] = (ints(case["masks"] + 1, rows) - 1).to(torch.int32)  # -1: no grammar
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    if case["op"] == "norm":
        state = _prepare_norm(case, make)
    elif case["op"] == "linear":
        state = _prepare_linear(case, make)
    else:
        state = _prepare_rules(case, make, gen)
    return dict(state, case=dict(case))


# ------------------------------------------------------------------ plain forms

def _plain_norm(s):
    """h = x + residual in the stream's type; its norm; e4m3 with a scale per row and 128 columns."""
    x, kind = s["x"], s["case"]["norm"]
    eps = 1e-5 if kind == "layer" else 1e-8
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    y = h.float()
    if kind == "rms":
        y = y * (1.0 / torch.sqrt((y * y).mean(1, keepdim=True) + eps)) * s["weight"]
    elif kind == "layer":
        y = y - y.mean(1, keepdim=True)
        y = y * (1.0 / torch.sqrt((y * y).mean(1, keepdim=True) + eps)) * s["weight"] + s["bias"]
    rows, k = y.shape
    kb = _blocks(k)
    y = torch.nn.functional.pad(y, (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    a = y.abs().amax(2).clamp_min(TINY)
    q = (y * (448.0 / a)[:, :, None]).clamp(-448, 448).to(E4M3).view(rows, kb * BLOCK)[:, :k]
    out = {"q": q, "scales": (a / 448.0).t().contiguous()}
    if s["residual"] is not None:
        out["sum"] = h
    return out


def _plain_linear(s):
    """Both operands as the values they stand for, one product in 32 bits, one rounding."""
    rows, k = s["q"].shape
    n = s["weight"].shape[0]
    x = s["q"].float() * s["scales"].t().repeat_interleave(BLOCK, 1)[:, :k]
    w = s["weight"].float() * s["weight_scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ w.t()
    return (y if s["bias"] is None else y + s["bias"]).to(s["out"])


def _plain_rules(s):
    """Penalties by each token's count, the biases, the grammar, the first largest token."""
    rows, vocab = s["logits"].shape
    l = s["logits"].float()
    dev = l.device
    if "history" in s:
        cap = s["history"].shape[1]
        valid = (torch.arange(cap, device=dev) < s["lengths"][:, None]).float()
        count = torch.zeros(rows, vocab, device=dev).scatter_add_(1, s["history"].long(), valid)
        rep = s["repetition"][:, None]
        punished = torch.where(l > 0, l / rep, l * rep) - (s["frequency"][:, None] * count + s["presence"][:, None])
        l = torch.where(count > 0, punished, l)
    if "dense_bias" in s:
        l = l + s["dense_bias"]
    if "bias_ids" in s:
        l = l + torch.zeros(rows, vocab, device=dev).scatter_(1, s["bias_ids"].long(), s["bias_values"])
    if "masks" in s:
        bits = ((s["masks"][:, :, None] >> torch.arange(32, device=dev, dtype=torch.int32)) & 1).bool().flatten(1)[:, :vocab]
        banned = ~bits[s["mask_rows"].clamp_min(0).long()] & (s["mask_rows"] >= 0)[:, None]
        l = l.masked_fill(banned, -math.inf)
    top = l.amax(1, keepdim=True)
    first = torch.where(l == top, torch.arange(vocab, device=dev), vocab).amin(1)
    tokens = torch.where(top[:, 0] > -math.inf, first, -1).to(torch.int32)
    return {"logits": l.to(s["logits"].dtype), "tokens": tokens}


# ------------------------------------------------------------------ one pass

def run(state):
    op = state["case"]["op"]
    if own:
        svl = _svl()
        if op == "norm":
            kind = state["case"]["norm"]
            q, scales, h = svl.add_norm_f8(state["x"], state["residual"], None if kind == "none" else kind, state["weight"],
                                           state["bias"], eps=1e-5 if kind == "layer" else 1e-8)
            return {"q": q, "scales": scales} if state["residual"] is None else {"q": q, "scales": scales, "sum": h}
        if op == "linear":
            return state["linear"](state["q"], state["scales"], out_dtype=state["out"])
        rules = {name: state[name] for name in ("history", "lengths", "repetition", "frequency", "presence", "dense_bias", "bias_ids",
                                                "bias_values", "masks", "mask_rows") if name in state}
        logits, tokens = svl.logits_rules(state["logits"], **rules)
        return {"logits": logits, "tokens": tokens}
    if op == "norm":
        return _plain_norm(state)
    if op == "linear":
        return _plain_linear(state)
    return _plain_rules(state)


def work(case):
    if case["op"] == "norm":
        rows, k, el = case["rows"], case["k"], 4 if case["dtype"] == "f32" else 2
        stream = el * rows * k * (3 if case["residual"] else 1)
        return {"bytes": stream + rows * k + 4 * rows * _blocks(k) + 4 * k * ("none", "rms", "layer").index(case["norm"]), "flops": 8 * rows * k}
    if case["op"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        scales = 4 * _blocks(k) * (rows + _blocks(n))
        return {"bytes": rows * k + n * k + scales + rows * n * (4 if case["out"] == "f32" else 2) + (4 * n if case["bias"] else 0), "flops": 2 * rows * n * k}
    rows, vocab, el = case["rows"], case["vocab"], 4 if case["dtype"] == "f32" else 2
    other = 4 * rows * case["history"] + 8 * rows * case["biased"] + (4 * vocab if case["dense"] else 0) + 4 * case["masks"] * -(-vocab // 32)
    return {"bytes": 2 * el * rows * vocab + other + 4 * rows, "flops": 6 * rows * vocab}


# ------------------------------------------------------------------ 64 bits

def _round_e4m3(v):
    """The nearest e4m3 value (ties to even): steps of 2^(e-3) for |v| in [2^e, 2^(e+1)), e at least -6."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_norm(s):
    case = s["case"]
    h = s["x"]
    if s["residual"] is not None:
        h = (h.double() + s["residual"].double()).to(h.dtype)
    v = h.double()
    if case["norm"] == "rms":
        v = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-8) * s["weight"].double()
    if case["norm"] == "layer":
        v = (v - v.mean(1, keepdim=True)) / torch.sqrt(v.var(1, unbiased=False, keepdim=True) + 1e-5) * s["weight"].double() + s["bias"].double()
    parts, scales = [], []
    for c in range(0, case["k"], BLOCK):
        g = v[:, c:c + BLOCK]
        top = torch.clamp(g.abs().max(1).values, min=TINY)
        parts.append(_round_e4m3(g * 448 / top[:, None]))
        scales.append(top / 448)
    out = {"q": torch.cat(parts, 1), "scales": torch.stack(scales)}
    if s["residual"] is not None:
        out["sum"] = h.double()
    return out


def _exact_linear(s):
    case = s["case"]
    y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device="cuda")
    for j, c in enumerate(range(0, case["k"], BLOCK)):
        part = s["q"][:, c:c + BLOCK].double() @ s["weight"][:, c:c + BLOCK].double().t()
        y += part * s["scales"][j].double()[:, None] * s["weight_scales"][:, j].double().repeat_interleave(BLOCK)[:case["n"]]
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_rules(s):
    case = s["case"]
    rows, vocab = case["rows"], case["vocab"]
    l = s["logits"].double()
    for r in range(rows):
        if "history" in s:
            said = s["history"][r, :min(int(s["lengths"][r]), case["history"])].long()
            ids, n = said.unique(return_counts=True)
            v = l[r, ids]
            rep = s["repetition"][r].double()
            l[r, ids] = torch.where(v > 0, v / rep, v * rep) - s["frequency"][r].double() * n - s["presence"][r].double()
        if "dense_bias" in s:
            l[r] += s["dense_bias"].double()
        if "bias_ids" in s:
            l[r, s["bias_ids"][r].long()] += s["bias_values"][r].double()
        if "masks" in s and int(s["mask_rows"][r]) >= 0:
            words = s["masks"][int(s["mask_rows"][r])]
            at = torch.arange(vocab, device=words.device)
            l[r, (words[at // 32] >> (at % 32)) & 1 == 0] = -math.inf
    # The token depends on a comparison of rounded values: it has no value in 64 bits.
    return {"logits": l, "tokens": None}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "linear":
        return _exact_linear(s)
    return _exact_rules(s)
