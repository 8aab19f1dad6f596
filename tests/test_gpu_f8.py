"""e4m3 rows and products on the GPU against plain forms in 64 bits.

Bounds, with u = 2^-24 (f32) per rounding:
  - a sum of k squares, whatever its order, is off by at most k u relative; the kernels add
    at most k / 256 + 32 of them in a chain, and a handful of roundings follow (root, division,
    two products), so y is within (k / 256 + 64) u of the formula, relative to the largest
    magnitude that enters it;
  - e4m3 rounds by at most half a step: 2^-4 of the value, or 2^-10 below the normal range;
  - a product sums k exact products and kblocks scaled partial sums. Each of those additions, and
    the scales' products, is off by at most 2 u of the magnitudes summed so far (2 u covers
    truncation as well as rounding): (k + 2 kblocks + 4) 2 u sum |x| |w|, and half a step of the
    output's type.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -100


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def norm_reference(h, norm, w, b, eps):
    """The norm of rows h (float64), and the bound on a kernel's deviation from it."""
    k = h.shape[1]
    slack = (k / 256 + 64) * U
    if norm is None:
        return h, np.zeros_like(h)
    c = h - (h.mean(1, keepdims=True) if norm == "layer" else 0.0)
    r = 1.0 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
    # The centred values carry the mean's rounding: relative to the row's largest magnitude.
    size = np.abs(h).max(1, keepdims=True) if norm == "layer" else np.abs(c)
    y, bound = c * r * w, slack * size * r * np.abs(w) + slack * np.abs(c * r * w)
    if norm == "layer":
        # r moves with the variance, whose terms move with the mean.
        bound = bound + slack * np.abs(c * r * w) * (np.abs(h).max(1, keepdims=True) * r)
        y, bound = y + b, bound + U * np.abs(y + b)
    return y, bound


def check_norm(q, scales, y, bound):
    """q and scales stand for y: the scale is the block's largest magnitude / 448 and every value
    within half a step."""
    rows, k = y.shape
    kb = -(-k // 128)
    assert q.shape == (rows, k) and scales.shape == (kb, rows)
    for b in range(kb):
        part, lim = y[:, b * 128:(b + 1) * 128], bound[:, b * 128:(b + 1) * 128]
        top = np.maximum(np.abs(part).max(1), TINY)
        s = scales[b].astype(np.float64)
        np.testing.assert_array_less(np.abs(s * 448 - top), lim.max(1) + 4 * U * top)
        v = part / s[:, None]
        got = q[:, b * 128:(b + 1) * 128]
        assert np.all(np.abs(got) <= 448)
        half = np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10) + lim / s[:, None] + 4 * U * np.abs(v)
        worst = np.abs(got - v) - half
        assert worst.max() <= 0, (b, worst.max())


def run_norm(rows, k, dtype, norm, residual, seed=0, strides=0, weight=True, scale=1.0):
    import torch

    import svl
    g = torch.Generator().manual_seed(seed)
    t = torch_dtype(dtype)
    x = (scale * torch.randn(rows, k + strides, generator=g)).to(t)[:, strides:]
    res = (scale * torch.randn(rows, k + 2 * strides, generator=g)).to(t)[:, :k] if residual else None
    w = 1 + 0.2 * torch.randn(k, generator=g) if norm and weight else None
    b = 0.3 * torch.randn(k, generator=g) if norm == "layer" and weight else None
    eps = 1e-5 if norm == "layer" else 1e-8
    dev = lambda a: None if a is None else a.cuda() if a.is_contiguous() else a.cuda().clone(memory_format=torch.preserve_format)  # noqa: E731
    xd = torch.empty(rows, k + strides, dtype=t, device="cuda")[:, strides:].copy_(x)
    rd = None if res is None else torch.empty(rows, k + 2 * strides, dtype=t, device="cuda")[:, :k].copy_(res)
    q, scales, h = svl.add_norm_f8(xd, rd, norm, dev(w), dev(b), eps=eps)
    want = x if res is None else (x.float() + res.float()).to(t)
    if res is not None:
        assert torch.equal(h.cpu(), want), "the sum is rounded once, as its type"
    h64 = want.double().numpy()
    one, zero = np.ones(k), np.zeros(k)
    y, bound = norm_reference(h64, norm, one if w is None else w.double().numpy(), zero if b is None else b.double().numpy(), eps)
    check_norm(q.float().cpu().numpy(), scales.cpu().numpy(), y, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("norm", ["rms", "layer", None])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 16), (5, 127), (2, 128), (7, 129), (1, 2048), (33, 2560), (4, 5637), (300, 1000), (2, 16384),
                                    (3, 32768), (5, 32761)])
def test_norm(svl_lib, dtype, norm, rows, k):
    run_norm(rows, k, dtype, norm, residual=True, seed=rows * 7 + k)
    run_norm(rows, k, dtype, norm, residual=False, seed=rows * 5 + k, weight=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("strides", [1, 3, 8, 20])
def test_norm_strides(svl_lib, dtype, strides):
    """Rows that start off every alignment, their neighbours left alone."""
    run_norm(9, 1000, dtype, "rms", True, strides=strides)
    run_norm(9, 1024, dtype, "layer", True, strides=strides)


def test_norm_range(svl_lib):
    """Values near the type's ends: blocks of zeros, denormals and huge values."""
    import torch

    import svl
    x = torch.zeros(4, 512, device="cuda")
    x[0, 130] = 1e-42
    x[1, :] = 3e38
    x[2, 5] = -7.0
    q, s, h = svl.add_norm_f8(x, norm=None)
    assert h is x
    assert torch.equal(s[0, [0, 3]], torch.full((2,), 2.0 ** -100 / 448, device="cuda")) and not q.float()[3].any()
    assert q.float()[0].abs().max() == 0  # far below the least scale
    assert torch.all(q.float()[1] == 448) and torch.allclose(s[:, 1] * 448, torch.tensor(3e38, device="cuda"))
    assert q.float()[2, 5] == -448 and q.float()[2].count_nonzero() == 1


def test_norm_not_finite(svl_lib):
    """A block that holds a NaN or an infinity stands for NaN; other rows and blocks do not change."""
    import torch

    import svl
    x = torch.randn(3, 300, device="cuda")
    clean = svl.add_norm_f8(x, norm=None)
    y = x.clone()
    y[1, 5], y[2, 290] = float("inf"), float("nan")
    q, s, _ = svl.add_norm_f8(y, norm=None)
    v = q.float() * s.t().repeat_interleave(128, 1)[:, :300]
    assert torch.isnan(v[1, :128]).all() and torch.isnan(v[2, 256:]).all()
    keep = torch.ones(3, 300, dtype=torch.bool)
    keep[1, :128] = keep[2, 256:] = False
    assert torch.equal(q.float().cpu()[keep], clean[0].float().cpu()[keep])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_in_place(svl_lib, dtype):
    """The sum may replace x or the residual."""
    import torch

    import svl
    x, r = (torch.randn(17, 2048, device="cuda").to(torch_dtype(dtype)) for _ in range(2))
    q, s, h = svl.add_norm_f8(x, r)
    for target in ("x", "r"):
        a, b = x.clone(), r.clone()
        q2, s2, h2 = svl.add_norm_f8(a, b, out_sum=a if target == "x" else b)
        assert torch.equal(h2, h) and torch.equal(s2, s) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8))
        assert torch.equal(b if target == "x" else a, r if target == "x" else x)


def quantised(rows, k, n, seed, bias=False, pad=0):
    """Random e4m3 rows and weights with block scales, on the GPU."""
    import torch
    g = torch.Generator().manual_seed(seed)
    f8 = torch.float8_e4m3fn
    ld = -(-k // 16) * 16 + 16 * pad
    # Bytes past k are NaN codes: nothing may read them.
    store = torch.full((max(rows, 1), ld), 0x7F, dtype=torch.uint8).view(f8)
    store[:, :k] = (100 * torch.randn(max(rows, 1), k, generator=g)).clamp(-448, 448).to(f8)
    kb, nb = -(-k // 128), -(-n // 128)
    return dict(q=store.cuda()[:rows, :k], s=(torch.rand(kb, rows, generator=g) * 0.02).cuda(),
                w=(100 * torch.randn(n, k, generator=g)).clamp(-448, 448).to(f8).cuda(),
                ws=(torch.rand(nb, kb, generator=g) * 0.001).cuda(), b=torch.randn(n, generator=g).cuda() if bias else None)


def linear_reference(d):
    x = d["q"].double() * d["s"].double().t().repeat_interleave(128, 1)[:, :d["q"].shape[1]]
    w = d["w"].double() * d["ws"].double().repeat_interleave(128, 0)[:d["w"].shape[0]].repeat_interleave(128, 1)[:, :d["w"].shape[1]]
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if d["b"] is not None:
        y, size = y + d["b"].double(), size + d["b"].double().abs()
    return y, size


def check_linear(got, d, out):
    import torch
    y, size = linear_reference(d)
    k = d["q"].shape[1]
    bound = (k + 2 * -(-k // 128) + 4) * 2 * U * size + torch.finfo(torch_dtype(out)).eps / 2 * y.abs()
    worst = ((got.double() - y).abs() / bound.clamp_min(1e-300)).max().item() if y.numel() else 0.0
    assert worst <= 1, worst


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,k", [
    (1, 1, 1), (1, 8, 16), (2, 100, 130), (1, 2048, 2048), (1, 8000, 2048), (15, 4001, 1000), (16, 256, 5632), (17, 129, 128), (31, 384, 640),
    (33, 1000, 2560), (64, 6144, 2048), (65, 512, 2047), (127, 130, 257), (128, 128, 128), (129, 2048, 5632), (255, 4001, 333),
    (256, 11264, 2048), (257, 640, 1024), (515, 4001, 2500), (1000, 2048, 10240), (2049, 1111, 999), (1500, 4001, 700), (8191, 2300, 300), (4000, 2560, 2048)])
def test_linear(svl_lib, rows, n, k, out):
    import svl
    d = quantised(rows, k, n, rows + n + k, bias=(rows + n) % 2 == 0)
    lin = svl.F8Linear(d["w"], d["ws"], d["b"])
    check_linear(lin(d["q"], d["s"], out_dtype=torch_dtype(out)), d, out)
    lin.check()


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(256, 1024, 6400), (300, 1000, 5000), (140, 1200, 2900), (147, 225, 2048), (290, 130, 700), (1000, 300, 300)])
def test_linear_few_tiles(svl_lib, rows, n, k, out):
    """More than 64 rows with few tiles, small ones and those that CTAs share; two runs give the same bits."""
    import torch

    import svl
    d = quantised(rows, k, n, rows + k, bias=True)
    lin = svl.F8Linear(d["w"], d["ws"], d["b"])
    got = lin(d["q"], d["s"], out_dtype=torch_dtype(out))
    check_linear(got, d, out)
    assert torch.equal(got, lin(d["q"], d["s"], out_dtype=torch_dtype(out)))


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_linear_padded(svl_lib, rows):
    """Rows with NaN codes between them, scales in a wider table, outputs in a wider table whose
    other columns and rows stay as they were; two runs give the same bits."""
    import torch

    import svl
    d = quantised(rows, 1000, 777, 3, bias=True, pad=2)
    wide = torch.full((8, rows + 5), float("nan"), device="cuda")
    wide[:, :rows] = d["s"]
    lin = svl.F8Linear(d["w"], d["ws"], d["b"])
    big = torch.full((rows + 2, 900), -1.0, device="cuda")
    got = lin(d["q"], wide[:, :rows], out=big[1:rows + 1, 50:827])
    check_linear(got, d, "f32")
    outside = big.clone()
    outside[1:rows + 1, 50:827] = -1.0
    assert torch.all(outside == -1.0)
    assert torch.equal(got, lin(d["q"], d["s"]))


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(100, 131, 8200), (128, 4001, 2500), (129, 257, 2600), (65, 135, 6000), (130, 8, 5000), (300, 1031, 6000)])
def test_linear_odd_outputs(svl_lib, rows, n, k, out):
    """Outputs of an odd width at an odd offset, also where CTAs share a tile; nothing outside is written."""
    import torch

    import svl
    d = quantised(rows, k, n, rows + n, bias=True)
    lin = svl.F8Linear(d["w"], d["ws"], d["b"])
    big = torch.full((rows + 2, n + 6), -1.0, device="cuda", dtype=torch_dtype(out))
    got = lin(d["q"], d["s"], out=big[1:rows + 1, 5:5 + n])
    check_linear(got, d, out)
    outside = big.clone()
    outside[1:rows + 1, 5:5 + n] = -1.0
    assert torch.all(outside == -1.0)


def test_linear_quantise(svl_lib):
    """F8Linear.quantise's weights are within half an e4m3 step of the f32 ones."""
    import torch

    import svl
    g = np.random.default_rng(5)
    w = g.standard_normal((200, 300)).astype(np.float32)
    w[:128, 128:256] = 0
    lin = svl.F8Linear.quantise(w, np.arange(200, dtype=np.float32))
    # Rows that pick one column each read the matrix back.
    eye = torch.zeros(300, 304, device="cuda")
    eye[:, :300] = torch.eye(300, device="cuda")
    got = lin(eye.to(torch.float8_e4m3fn)[:, :300], torch.ones(3, 300, device="cuda")).t().cpu().numpy() - np.arange(200, dtype=np.float32)[:, None]
    for i in range(2):
        for j in range(3):
            blk = np.s_[i * 128:min(200, i * 128 + 128), j * 128:min(300, j * 128 + 128)]
            s = max(np.abs(w[blk]).max(), TINY) / 448
            # The bias was added and taken off again: u of it each time.
            half = np.maximum(np.abs(w[blk]) * 2.0 ** -4, s * 2.0 ** -10) * (1 + 8 * U) + 2 * U * 200
            assert np.all(np.abs(got[blk] - w[blk]) <= half), (i, j)


def test_linear_many_outputs(svl_lib):
    """More than 65,535 tiles of matrix rows."""
    import torch

    import svl
    n = 65536 * 128 + 5
    w = np.ones((n, 1), np.float32)
    w[::2] = -0.5
    lin = svl.F8Linear.quantise(w)
    q, s, _ = svl.add_norm_f8(torch.tensor([[3.0], [-8.0]], device="cuda"), norm=None)
    got = lin(q, s)
    # The row's and the matrix's scales round once each, the products twice.
    want = torch.tensor([[3.0], [-8.0]], device="cuda") * torch.from_numpy(w).cuda().t()
    assert torch.all((got - want).abs() <= want.abs() * 4 * 2.0 ** -24)


def test_linear_refuses(svl_lib):
    import torch

    import svl
    from svl._lib import SvlError
    d = quantised(4, 256, 128, 1)
    lin = svl.F8Linear(d["w"], d["ws"])
    with pytest.raises(ValueError, match="q must"):
        lin(d["q"][:, :128], d["s"])
    with pytest.raises(ValueError, match="scales must"):
        lin(d["q"], d["s"][:1])
    with pytest.raises(ValueError, match="out must"):
        lin(d["q"], d["s"], out=torch.empty(4, 127, device="cuda"))
    odd = torch.zeros(4, 257, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :256]
    with pytest.raises(SvlError, match="multiple of 16"):
        lin(odd, d["s"])
    with pytest.raises(SvlError, match="aligned"):
        lin(torch.zeros(4, 272, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, 8:264], d["s"])
    with pytest.raises(ValueError, match="scales must"):
        svl.F8Linear(d["w"], d["ws"][:, :1])
    assert lin(d["q"][:0], d["s"][:, :0]).shape == (0, 128)


def test_streams_and_graphs(svl_lib):
    """The same answers on another stream, from two calls at once on two streams, and from a captured
    graph replayed on new inputs."""
    import torch

    import svl
    x, r = torch.randn(40, 2048, device="cuda"), torch.randn(40, 2048, device="cuda")
    d = quantised(1, 2048, 6144, 9)
    lin = svl.F8Linear(d["w"], d["ws"])

    def step(a, b):
        q, s, h = svl.add_norm_f8(a, b)
        return lin(q, s), h

    want, want_h = step(x, r)
    other, other_h = step(r, x * 2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        got = [step(x, r) for _ in range(5)]
    with torch.cuda.stream(s2):
        got2 = [step(r, x * 2) for _ in range(5)]
    torch.cuda.synchronize()
    for y, h in got:
        assert torch.equal(y, want) and torch.equal(h, want_h)
    for y, h in got2:
        assert torch.equal(y, other) and torch.equal(h, other_h)
    a, b = x.clone(), r.clone()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = step(a, b)
    with torch.cuda.graph(graph2):
        y2, h2 = step(a, b)
    a.copy_(r)
    b.copy_(x * 2)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        graph.replay()
    with torch.cuda.stream(s2):
        graph2.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, other) and torch.equal(h, other_h) and torch.equal(y2, other)
    lin.check()


def test_outputs_belong_to_their_stream(svl_lib):
    """Outputs of a call on another stream are not given out again while that stream has yet to write them."""
    import torch

    import svl
    side = torch.cuda.Stream()
    x = torch.randn(64, 4096, device="cuda")
    lin = svl.F8Linear.quantise(np.ones((256, 4096), np.float32))
    q, s, _ = svl.add_norm_f8(x)
    lg = lin(q, s)
    for call in (lambda: svl.add_norm_f8(x, x, stream=side), lambda: lin(q, s, stream=side), lambda: svl.logits_rules(lg, stream=side)):
        for warm in (True, False):  # loading a kernel for the first time waits for the device
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                torch.cuda._sleep(100_000_000)
            got = call()
            sizes = [(t.shape, t.dtype) for t in (got if isinstance(got, tuple) else (got,)) if t is not x]
            del got
            taken = [torch.full(shape, 7.0, device="cuda").to(dtype) for shape, dtype in sizes for _ in range(2)]
            torch.cuda.current_stream().synchronize()
            waiting = not side.query()
            side.synchronize()
            assert all(torch.all(t.float() == 7.0) for t in taken)
        assert waiting, "the side stream had ended before the memory was taken"
    side.synchronize()
    if torch.cuda.device_count() > 1:
        with pytest.raises(ValueError, match="stream must"):
            svl.add_norm_f8(x, stream=torch.cuda.Stream(1))


def test_linear_closed_during_capture(svl_lib):
    """An F8Linear that goes away while a graph is captured (as the collector may decide) leaves the capture alone."""
    import torch

    import svl
    x = torch.randn(3, 256, device="cuda")
    lin, other = (svl.F8Linear.quantise(np.eye(256, dtype=np.float32)) for _ in range(2))
    q, s, _ = svl.add_norm_f8(x, norm=None)
    want = lin(q, s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q2, s2, _ = svl.add_norm_f8(x, norm=None)
        other.close()
        got = lin(q2, s2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k", [1, 5, 33, 511, 513, 1025, 2561, 4097, 5637, 8191, 9001, 16385])
def test_norm_odd_rows(svl_lib, dtype, k):
    """Rows of every alignment, x, residual and sum differently, with what lies around the sum's rows
    left as it was; in place too."""
    import torch

    import svl
    t = torch_dtype(dtype)
    g = torch.Generator(device="cuda").manual_seed(k)
    rows = 19
    for off, (a, b, c) in enumerate([(0, 0, 0), (1, 0, 3), (0, 7, 1), (3, 3, 3), (5, 2, 8), (8, 8, 0)]):
        wide = lambda o: torch.randn(rows, k + o + off % 3, device="cuda", generator=g).to(t)  # noqa: E731
        x, r, big = wide(a)[:, a:a + k], wide(b)[:, b:b + k], torch.full((rows, k + c + off % 2), 9.0, device="cuda", dtype=t)
        want_h = (x.float() + r.float()).to(t)
        want_q, want_s, _ = svl.add_norm_f8(want_h.contiguous() if k % 8 == 0 else torch.nn.functional.pad(want_h, (0, -k % 16))[:, :k], norm=None)
        q, s, h = svl.add_norm_f8(x, r, norm=None, out_sum=big[:, c:c + k])
        assert torch.equal(h, want_h) and torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
        around = big.clone()
        around[:, c:c + k] = 9.0
        assert torch.all(around == 9.0)
        q, s, h = svl.add_norm_f8(x, r, norm=None, out_sum=x)
        assert torch.equal(h, want_h) and torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
