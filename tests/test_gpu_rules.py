"""The rules between logits and token on the GPU against a plain numpy form that rounds where the
rules say (f32 after each operation): values and tokens are identical."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F = np.float32


def reference(logits, r):
    """logits f32 [rows, vocab]; r: the rules as numpy arrays. Returns (logits, tokens, history, lengths)."""
    rows, vocab = logits.shape
    out = logits.astype(F).copy()
    tokens = np.full(rows, -1, np.int32)
    hist = None if r.get("history") is None else r["history"].copy()
    lens = None if r.get("lengths") is None else r["lengths"].copy()
    first = r.get("first_penalised", 0)
    with np.errstate(all="ignore"):
        for i in range(rows):
            l = out[i]
            if hist is not None:
                said = hist[i, :min(max(lens[i], 0), hist.shape[1])]
                said = said[(said >= first) & (said >= 0) & (said < vocab)]
                ids, n = np.unique(said, return_counts=True)
                rep = F(1) if r.get("repetition") is None else r["repetition"][i]
                freq = F(0) if r.get("frequency") is None else r["frequency"][i]
                pres = F(0) if r.get("presence") is None else r["presence"][i]
                v = l[ids]
                v = np.where(v > 0, v / rep, v * rep).astype(F)
                l[ids] = v - ((freq * n.astype(F)).astype(F) + pres).astype(F)
            if r.get("dense_bias") is not None:
                l[:] = l + r["dense_bias"]
            if r.get("bias_ids") is not None:
                for j, v in zip(r["bias_ids"][i], r["bias_values"][i]):
                    if 0 <= j < vocab:
                        l[j] = l[j] + v
            if r.get("masks") is not None:
                m = i if r.get("mask_rows") is None else r["mask_rows"][i]
                if 0 <= m < r["masks"].shape[0]:
                    at = np.arange(vocab)
                    ok = (r["masks"][m].view(np.uint32)[at // 32] >> (at % 32).astype(np.uint32)) & 1
                    l[ok == 0] = -np.inf
            c = np.where(np.isnan(l), -np.inf, l)
            if c.max() > -np.inf:
                tokens[i] = int(np.argmax(c))
            if r.get("append") and hist is not None and tokens[i] >= max(first, 0):
                n = max(int(lens[i]), 0)
                hist[i, n % hist.shape[1]] = tokens[i]
                lens[i] = n + 1
    return out, tokens, hist, lens


def make(rows, vocab, seed, history=0, biased=0, dense=False, masks=0, pads=False):
    g = np.random.default_rng(seed)
    r = {}
    if history:
        r["history"] = np.where(g.random((rows, history)) < 0.6, g.integers(0, min(vocab, 9), (rows, history)),
                                g.integers(0, vocab, (rows, history))).astype(np.int32)
        if pads:
            r["history"][g.random((rows, history)) < 0.2] = -1
            r["history"][g.random((rows, history)) < 0.1] = vocab + 3
        r["lengths"] = g.integers(0, 2 * history + 1, rows).astype(np.int32)
        r["lengths"][::3] = history
        r["repetition"] = (1 + g.random(rows)).astype(F)
        r["frequency"] = g.random(rows).astype(F)
        r["presence"] = g.random(rows).astype(F)
    if biased:
        r["bias_ids"] = g.integers(-1 if pads else 0, vocab + (2 if pads else 0), (rows, biased)).astype(np.int32)  # some twice
        r["bias_values"] = (3 * g.standard_normal((rows, biased))).astype(F)
    if dense:
        r["dense_bias"] = g.standard_normal(vocab).astype(F)
    if masks:
        r["masks"] = g.integers(-2 ** 31, 2 ** 31, (masks, -(-vocab // 32) + (1 if pads else 0))).astype(np.int32)
        r["mask_rows"] = g.integers(-1, masks + (1 if pads else 0), rows).astype(np.int32)
    return g, r


def run(logits, r, dtype="f32", offset=0, in_place=False):
    """The rules on the GPU; logits numpy f32. Rows `offset` elements off their alignment."""
    import torch

    import svl
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    rows, vocab = logits.shape
    x = torch.empty(rows, vocab + offset, dtype=t, device="cuda")[:, offset:]
    x.copy_(torch.from_numpy(logits))
    dev = {k: torch.from_numpy(v.copy()).cuda() if isinstance(v, np.ndarray) else v for k, v in r.items()}
    out, tok = svl.logits_rules(x, **dev, out=x if in_place else None)
    if not in_place:
        assert torch.equal(x.cpu(), torch.from_numpy(logits).to(t)) or np.isnan(logits).any()
    return out.float().cpu().numpy(), tok.cpu().numpy(), dev


def check(logits, r, dtype="f32", **kw):
    import torch
    if dtype == "bf16":
        logits = torch.from_numpy(logits).bfloat16().float().numpy()
    want, tokens, hist, lens = reference(logits, r)
    got, tok, dev = run(logits, r, dtype, **kw)
    if dtype == "bf16":
        want = torch.from_numpy(want).bfloat16().float().numpy()
    np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(tok, tokens)
    if r.get("append"):
        np.testing.assert_array_equal(dev["history"].cpu().numpy(), hist)
        np.testing.assert_array_equal(dev["lengths"].cpu().numpy(), lens)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (3, 33), (2, 4095), (5, 4001), (1, 8000), (2, 8193), (40, 2049), (3, 50257), (1, 131072),
                                        (300, 1000)])
def test_rules(svl_lib, dtype, rows, vocab):
    for n, kw in enumerate([dict(), dict(history=50), dict(biased=20), dict(dense=True), dict(masks=2),
                            dict(history=300, biased=70, dense=True, masks=3, pads=True)]):
        g, r = make(rows, vocab, 100 * n + rows + vocab, **kw)
        logits = (4 * g.standard_normal((rows, vocab))).astype(F)
        check(logits, r, dtype, offset=n % 4)


@pytest.mark.parametrize("rows,vocab,history,biased", [(2, 200, 65535, 0), (2, 70000, 5000, 4000), (1, 40, 100, 65535)])
def test_long_lists(svl_lib, rows, vocab, history, biased):
    g, r = make(rows, vocab, 5, history=history, biased=biased, pads=True)
    if biased == 65535:
        r["bias_values"] = (r["bias_values"] * 0.01).astype(F)
    check((4 * g.standard_normal((rows, vocab))).astype(F), r)


def test_one_token_everywhere(svl_lib):
    """The same index in every history and bias slot: the count is the history's length, the
    biases add up in order."""
    g, r = make(3, 5000, 8, history=60000, biased=3000)
    r["history"][:] = 4321
    r["lengths"][:] = [60000, 0, 17]
    r["bias_ids"][:] = 4321
    check((4 * g.standard_normal((3, 5000))).astype(F), r)


def test_ties_and_nothing_left(svl_lib):
    """Equal values: the lowest index; -0 and 0 are equal; NaN and -infinity are never picked; a
    row whose grammar leaves nothing has no token; the type's lowest value still is a value."""
    low = np.finfo(F).min
    l = np.zeros((8, 300), F)
    l[0, :] = 2.5
    l[1, :] = -1
    l[1, [77, 200]] = [-0.0, 0.0]
    l[2, :] = np.nan
    l[2, 123] = -5
    l[3, :] = -np.inf
    l[4, :] = low
    l[5, :] = np.nan
    l[6, :] = np.inf
    l[7, 250:] = 1
    check(l, {})
    masks = np.full((2, 10), -1, np.int32)
    masks[1] = 0
    check(l, {"masks": masks, "mask_rows": np.array([1, 0, 1, 0, -1, 5, 0, 0], np.int32)})
    out, tok, _ = run(l, {"masks": masks, "mask_rows": np.ones(8, np.int32)})
    assert np.all(tok == -1) and np.all(np.isneginf(out))
    check(l, {"masks": np.full((8, 10), 1 << 3, np.int32)})  # row r takes mask r: tokens 3, 35, ...
    check(l, {"dense_bias": np.full(300, low, F)})


@pytest.mark.parametrize("rows,vocab", [(1, 8000), (9, 4001), (200, 130), (2, 131072)])
def test_append(svl_lib, rows, vocab):
    """The picked tokens are recorded: rings that wrap, lengths of zero, ids below the first
    penalised one neither counted nor recorded; a full ring of the same graph's picks."""
    import torch

    import svl
    g, r = make(rows, vocab, 11, history=7, biased=3, masks=2)
    r["masks"][1] = 0
    r["append"] = True
    for first in (0, vocab // 2):
        r["first_penalised"] = first
        check((4 * g.standard_normal((rows, vocab))).astype(F), r)
        check((4 * g.standard_normal((rows, vocab))).astype(F), r, in_place=True)
    # Eight steps by a replayed graph against eight steps of the plain form.
    r["lengths"][:] = 0
    r["first_penalised"] = 3
    steps = [(4 * g.standard_normal((rows, vocab))).astype(F) for _ in range(8)]
    x = torch.empty(rows, vocab, device="cuda")
    dev = {k: torch.from_numpy(v.copy()).cuda() if isinstance(v, np.ndarray) else v for k, v in r.items()}
    graph = torch.cuda.CUDAGraph()
    x.copy_(torch.from_numpy(steps[0]))
    with torch.cuda.graph(graph):
        out, tok = svl.logits_rules(x, **dev)
    for l in steps:
        x.copy_(torch.from_numpy(l))
        graph.replay()
        want, tokens, r["history"], r["lengths"] = reference(l, r)
        np.testing.assert_array_equal(tok.cpu().numpy(), tokens)
        np.testing.assert_array_equal(out.cpu().numpy(), want)
    np.testing.assert_array_equal(dev["history"].cpu().numpy(), r["history"])


def test_history_count_near_its_end(svl_lib):
    """Lengths up to 2^31 - 1: the ring goes on at the next slot."""
    import torch

    import svl
    h = torch.full((2, 10), 5, dtype=torch.int32, device="cuda")
    n = torch.tensor([2 ** 31 - 2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    l = torch.zeros(2, 64, device="cuda")
    l[:, 9] = 1
    for step in range(3):
        svl.logits_rules(l, history=h, lengths=n, append=True)
    for row, start in ((0, 2 ** 31 - 2), (1, 2 ** 31 - 1)):
        want = [5] * 10
        for s in range(3):
            want[(start + s) % 10] = 9
        assert h[row].tolist() == want and n[row] >= 10


def test_only_tokens_or_only_logits(svl_lib):
    """Through the C ABI: tokens without logits kept, logits without tokens, and no rules at all."""
    import torch

    from svl._lib import check as ok, lib
    l = torch.randn(6, 1000, device="cuda")
    tok, out = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros_like(l)
    torch.cuda.synchronize()
    ok(lib().svl_logits_rules_device(0, 6, 1000, 0, l.data_ptr(), 1000, None, None, 0, tok.data_ptr(), None))
    ok(lib().svl_logits_rules_device(0, 6, 1000, 0, l.data_ptr(), 1000, None, out.data_ptr(), 1000, None, None))
    torch.cuda.synchronize()
    assert torch.equal(out, l) and torch.equal(tok.long(), l.argmax(1))


@pytest.mark.parametrize("rows,vocab,history,biased,dtype", [
    (1, 140000, 9000, 300, "f32"),     # two chunks per CTA, lists too long for a slot each in one
    (1, 1100001, 700, 5, "bf16"),      # chunks without room for a whole eighth
    (150, 20001, 60, 9, "bf16"),       # more rows than SMs
    (300, 16390, 2100, 0, "f32"),      # history entries past the first in flight
    (33, 131072, 40, 8, "bf16"),
    (120, 17001, 50, 9, "f32")])       # two CTAs per SM
@pytest.mark.parametrize("in_place", [False, True])
def test_splits_and_chunks(svl_lib, rows, vocab, history, biased, dtype, in_place):
    g, r = make(rows, vocab, rows + vocab, history=history, biased=biased, dense=True, masks=2)
    check((4 * g.standard_normal((rows, vocab))).astype(F), r, dtype, offset=rows % 8, in_place=in_place)


def test_edges_of_rows(svl_lib):
    """The best token at each end of rows that start off their alignment, touched or not, and no
    other token left in between."""
    for vocab in (1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 33):
        for offset in range(8):
            for at in {0, vocab - 1, vocab // 2}:
                logits = np.zeros((3, vocab), F)
                logits[:, at] = 5
                r = {"history": np.full((3, 4), at, np.int32), "lengths": np.array([0, 1, 4], np.int32),
                     "frequency": np.full(3, 2, F), "presence": np.zeros(3, F), "repetition": np.ones(3, F)}
                for dtype in ("f32", "bf16"):
                    check(logits, r, dtype, offset=offset)
                    check(logits, {}, dtype, offset=offset, in_place=True)
