"""The 8-bit operators where their ordinary tests do not go: values in the middle of two e4m3 values."""
import numpy as np
import pytest

from test_gpu_f8 import TINY, torch_dtype

pytestmark = pytest.mark.gpu

F = np.float32


def nearest_e4m3(v):
    """The nearest e4m3 value of v (float64, |v| <= 448), ties to even."""
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -20))), -6)
    step = 2.0 ** (e - 3)
    return np.rint(v / step) * step


def quantised(y):
    """Rows y (float64) as (q, scales [kblocks, rows]), from y * 448 / a in 64 bits.

    Of values y and a with 8 significant bits the quotient is 7 Y / T * 2^n with whole Y, T < 2^8: it is a middle
    (5 bits) or at least 2^-14 of itself away from one, and a middle has a float64. So q is the nearest value of
    the exact quotient."""
    q, s = [], []
    for c in range(0, y.shape[1], 128):
        part = y[:, c:c + 128]
        top = np.maximum(np.abs(part).max(1), TINY)
        q.append(nearest_e4m3(part * 448 / top[:, None]))
        s.append(top / 448)
    return np.concatenate(q, 1), np.stack(s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,residual", [(333, 5637, False), (200, 1000, True), (64, 200, False), (3, 20000, False), (2, 32768, True)])
def test_rows_of_few_bits_take_the_nearest(svl_lib, dtype, rows, k, residual):
    """Values of 8 significant bits without a norm: many lie in the middle of two e4m3 values."""
    import torch

    import svl
    g = torch.Generator().manual_seed(rows + k)
    x, r = (torch.randn(rows, k, generator=g).bfloat16().cuda() for _ in range(2))
    if residual and dtype == "f32":
        r = r * 0  # the sum keeps its 8 bits
    t = torch_dtype(dtype)
    q, s, h = svl.add_norm_f8(x.to(t), r.to(t) if residual else None, None)
    want, scales = quantised(h.double().cpu().numpy())
    np.testing.assert_array_equal(q.double().cpu().numpy(), want)
    np.testing.assert_array_equal(s.cpu().numpy(), scales.astype(F))


def test_weights_of_few_bits_take_the_nearest(svl_lib):
    """F8Linear.quantise of a bf16 checkpoint's weights."""
    import torch

    import svl
    n, k = 600, 512
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(3)).bfloat16().float().numpy()
    lin = svl.F8Linear.quantise(w)
    # Rows that pick one column each read the matrix back: one product with the scale, rounded to f32.
    got = lin(torch.eye(k, device="cuda").to(torch.float8_e4m3fn), torch.ones(k // 128, k, device="cuda")).t().cpu().numpy()
    for i in range(0, n, 128):
        for j in range(0, k, 128):
            blk = w[i:i + 128, j:j + 128].astype(np.float64)
            top = np.abs(blk).max()
            np.testing.assert_array_equal(got[i:i + 128, j:j + 128], nearest_e4m3(blk * 448 / top).astype(F) * F(F(top) / F(448)))


def test_matrix_refuses_a_stream_of_another_device(svl_lib):
    """As the operators do: the copies would not wait for the work of the stream that was meant."""
    import types

    import torch

    import svl
    w, s = torch.zeros(128, 128, device="cuda").to(torch.float8_e4m3fn), torch.ones(1, 1, device="cuda")
    # What a stream of a second GPU looks like, its default one.
    elsewhere = types.SimpleNamespace(device=torch.device("cuda", torch.cuda.current_device() + 1), cuda_stream=0)
    with pytest.raises(ValueError, match="stream must be one of"):
        svl.F8Linear(w, s, stream=elsewhere)
    svl.F8Linear(w, s, stream=torch.cuda.Stream()).close()
