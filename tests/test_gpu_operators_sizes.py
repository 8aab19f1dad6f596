"""The 8-bit operators and the rules at their largest sizes: offsets past 2^31 elements, the longest axes."""
import numpy as np
import pytest

from test_gpu_f8 import check_linear, quantised, torch_dtype

pytestmark = pytest.mark.gpu


def same_bits(a, b):
    import torch
    ints = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.contiguous().view(ints), b.contiguous().view(ints))


@pytest.mark.parametrize("dtype,rows,k", [("bf16", 140001, 16000), ("f32", 70001, 32768), ("bf16", 300001, 7333)])
def test_norm_far_rows(svl_lib, dtype, rows, k):
    """Rows past 2^31 elements are as those of a small call."""
    import torch

    import svl
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.empty(rows, k, dtype=torch_dtype(dtype), device="cuda").normal_(generator=g)
    w = torch.ones(k, device="cuda").normal_(1, 0.1, generator=g)
    q, s, h = svl.add_norm_f8(x, x, "rms", w)
    for r in (0, rows // 2, rows - 40):
        part = x[r:r + 40].contiguous()
        q2, s2, h2 = svl.add_norm_f8(part, part, "rms", w)
        assert same_bits(q[r:r + 40], q2) and same_bits(s[:, r:r + 40], s2) and same_bits(h[r:r + 40], h2)


@pytest.mark.parametrize("out,rows,n,k", [("f32", 140001, 16000, 130), ("bf16", 140001, 16001, 256), ("bf16", 1100001, 130, 2048)])
def test_linear_far_rows(svl_lib, out, rows, n, k):
    """Outputs, and rows, past 2^31 elements."""
    import torch

    import svl
    small = quantised(4096, k, n, n + k, bias=True)
    times = -(-rows // 4096)
    ld = -(-k // 16) * 16
    q = torch.empty(times * 4096, ld, dtype=torch.uint8, device="cuda")
    q.view(times, 4096, ld)[:, :, :k] = small["q"].view(torch.uint8)
    q = q.view(torch.float8_e4m3fn)[:rows, :k]
    s = small["s"].repeat(1, times)[:, :rows].contiguous()
    lin = svl.F8Linear(small["w"], small["ws"], small["b"])
    got = lin(q, s, out_dtype=torch_dtype(out))
    lin.check()
    for r in (0, rows // 2 // 4096 * 4096, (times - 1) * 4096):
        m = min(4096, rows - r)
        check_linear(got[r:r + m], dict(small, q=small["q"][:m], s=small["s"][:, :m]), out)


@pytest.mark.parametrize("rows", [1, 31, 90, 300, 1000])
def test_linear_longest_axis(svl_lib, rows):
    """k = 2^20, 8,192 blocks."""
    import torch

    import svl
    d = quantised(rows, 1 << 20, 130, rows, bias=True)
    lin = svl.F8Linear(d["w"], d["ws"], d["b"])
    got = lin(d["q"], d["s"])
    lin.check()
    # In pieces: the reference's operands in 64 bits would take 8 bytes for each of ours.
    y, size = torch.zeros(rows, 130, dtype=torch.float64, device="cuda"), torch.zeros(rows, 130, dtype=torch.float64, device="cuda")
    for c in range(0, 1 << 20, 1 << 16):
        x = d["q"][:, c:c + (1 << 16)].double() * d["s"][c // 128:c // 128 + 512].double().t().repeat_interleave(128, 1)
        w = d["w"][:, c:c + (1 << 16)].double() * d["ws"][:, c // 128:c // 128 + 512].double().repeat_interleave(128, 0)[:130].repeat_interleave(128, 1)
        y += x @ w.t()
        size += x.abs() @ w.abs().t()
    y, size = y + d["b"].double(), size + d["b"].double().abs()
    # Each of the additions rounds by at most 2 u of the magnitudes so far.
    bound = ((1 << 20) + 2 * 8192 + 4) * 2 * 2.0 ** -24 * size + 2.0 ** -24 * y.abs()
    assert ((got.double() - y).abs() <= bound).all()
    # That bound is wide at this length. A block that is left out, 2^-13 of the magnitudes and about a tenth of it
    # after its own signs, is told at 2^-18, which roundings of either sign stay far below.
    assert ((got.double() - y).abs() <= 2.0 ** -24 * 64 * size).all()


def test_rules_far_rows(svl_lib):
    """Logits past 2^31 elements, with every rule, in place too: as the rows of a small call."""
    import torch

    import svl
    rows, vocab = 17001, 131071
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    ints = lambda high, *shape: torch.randint(0, high, shape, device="cuda", dtype=torch.int32, generator=g)  # noqa: E731
    r = dict(history=ints(vocab, rows, 50), lengths=ints(100, rows), repetition=torch.full((rows,), 1.5, device="cuda"),
             bias_ids=ints(vocab, rows, 9), bias_values=torch.randn(rows, 9, device="cuda", generator=g), mask_rows=ints(3, rows))
    shared = dict(masks=torch.randint(-2 ** 31, 2 ** 31, (3, 4096), device="cuda", generator=g).to(torch.int32),
                  dense_bias=torch.randn(vocab, device="cuda", generator=g))
    out, tokens = svl.logits_rules(logits, **r, **shared)
    for a in (0, rows // 2, rows - 5):
        o, t = svl.logits_rules(logits[a:a + 5], **{k: v[a:a + 5] for k, v in r.items()}, **shared)
        assert same_bits(out[a:a + 5], o) and torch.equal(tokens[a:a + 5], t)
    again, tokens2 = svl.logits_rules(logits, **r, **shared, out=logits)
    assert again is logits and torch.equal(tokens, tokens2)
    for a in range(0, rows, 1000):
        assert same_bits(out[a:a + 1000], logits[a:a + 1000])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rules_long_vocabulary(svl_lib, dtype):
    """A row of 300,000,001 tokens: many chunks per CTA, touched tokens in each."""
    import torch

    import svl
    vocab = 300_000_001
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.empty(1, vocab, dtype=torch_dtype(dtype), device="cuda").normal_(generator=g)
    said = torch.randint(0, vocab, (1, 4000), device="cuda", dtype=torch.int32, generator=g)
    said[0, :4] = torch.tensor([0, vocab - 1, vocab // 2, vocab - 1], dtype=torch.int32)
    ids = torch.randint(0, vocab, (1, 300), device="cuda", dtype=torch.int32, generator=g)
    ids[0, -2:] = torch.tensor([vocab - 2, vocab - 2], dtype=torch.int32)
    values = torch.full((1, 300), 1.0, device="cuda")
    values[0, -2:] = 8.0
    out, token = svl.logits_rules(logits, history=said, lengths=torch.full((1,), 4000, dtype=torch.int32, device="cuda"),
                                  presence=torch.full((1,), 0.5, device="cuda"), bias_ids=ids, bias_values=values)
    want = logits[0].float()
    seen = said[0].long().unique()
    want[seen] -= 0.5
    for i, v in zip(ids[0].tolist(), values[0].tolist()):
        want[i] += v
    assert token.item() == want.argmax().item() == vocab - 2
    assert torch.equal(out[0].float(), want.to(out.dtype).float())
