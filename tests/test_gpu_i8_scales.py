"""Products of the 8-bit integer path whose scales' product leaves f32's range, or its normal range, while the result is in it:
rows with a largest value of 2^-110 and below, results of zero between huge scales."""
import pytest
import torch

from coachwhip_amd import i8, ops

from .test_gpu_i8 import DTYPES, U, gen, half, rand_rows, randn, say

pytestmark = pytest.mark.gpu

# every kernel of the products: few rows (16, 32, 64), the rings (64 x 64, 64 x 128, 128 x 128) and 256 x 256
SHAPES = [(1, 100, 300), (3, 40, 1000), (20, 300, 640), (50, 300, 640), (129, 255, 896), (300, 1500, 1500), (512, 4001, 1500), (700, 4096, 640), (5000, 3001, 897),
          (8200, 8200, 100)]


def check(y, p, bias, dtype):
    """y is the exact value (the sum, its scales and the bias in 64 bits) but for three roundings of f32 where all scales are usual
    ones (the sum's conversion and the scales' product, of p; the sum with the bias) and its type's: subnormal steps count."""
    want = p if bias is None else p + bias.double()
    step = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[dtype]
    err = (y.double() - want).abs()
    own = half(dtype) if dtype != torch.float32 else 0
    assert (err <= (1 + 2.0 ** -20) * (2 * U * p.abs() + (U + own) * want.abs() + (step + 2.0 ** -149) / 2)).all(), float(err.max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products_of_tiny_rows(m, n, k, dtype):
    say("tiny rows", m, n, k, dtype)
    g = gen(m + n + k)
    (xq, xs), (wq, ws) = rand_rows(g, m, k), rand_rows(g, n, k)
    # rows of x from usual ones to a largest value of 2^-130; channels of w at usual scales, and two of others
    xs = xs * torch.tensor([1.0, 2.0 ** -104, 2.0 ** -111, 2.0 ** -118, 2.0 ** -130], device="cuda").repeat(m // 5 + 1)[:m]
    if m == 1:
        xs = xs * 2.0 ** -118
    ws = ws * 5e-4
    ws[::7] *= 2.0 ** -20
    ws[3::11] *= 2.0 ** 60
    p = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    fits = p.abs() < 60000 if dtype == torch.float16 else p.abs() < 1e38
    for bias in (None, randn(g, n) * 2.0 ** -105):
        y = i8.I8MatMul(i8.I8Matrix(wq, ws, k), bias)(i8.I8Rows(xq, xs, k), dtype)
        check(y.double()[fits], p[fits], None if bias is None else bias.expand_as(p)[fits], dtype)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_sums_of_zero_between_huge_scales(m, n, k):
    say("huge scales", m, n, k)
    g = gen(m)
    (xq, xs), (wq, ws) = rand_rows(g, m, k), rand_rows(g, n, k)
    xq[::2] = 0
    y = i8.I8MatMul(i8.I8Matrix(wq, ws * 2.0 ** 60, k))(i8.I8Rows(xq, xs * 2.0 ** 90, k))
    assert (y[::2] == 0).all()
    p = (xq.double() @ wq.double().t()) * (xs * 2.0 ** 90).double()[:, None] * (ws * 2.0 ** 60).double()
    y = i8.I8MatMul(i8.I8Matrix(wq, ws * 2.0 ** 60, k), randn(g, n))(i8.I8Rows(xq, xs * 2.0 ** 90, k))
    assert not torch.isnan(y).any() and (torch.isinf(y[1::2]) == (p[1::2].abs() > torch.finfo(torch.float32).max)).all()


@pytest.mark.parametrize("T", [1, 5, 1030])  # (in two launches, and grouped)
@pytest.mark.parametrize("gate,down", [(-80, -38), (-104, 20)])
def test_layer_of_tiny_scales(T, gate, down):
    """One expert whose hidden rows are 128 equal values g / 2 (u = 0 in the clamped form), with scales of about 2^-35 on x, 2^gate
    and 2^down: the product of the scales of down, or of gate, is subnormal and no result is."""
    say("layer of tiny scales", T, gate, down)
    H, I, g = 256, 128, gen(T)
    x = torch.randint(64, 128, (T, H), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(64, 128, (H,), generator=g, device="cuda", dtype=torch.int8)
    banks = [w.expand(1, I, H).contiguous(), torch.zeros(1, I, H, dtype=torch.int8, device="cuda"), torch.full((1, H, I), 127, dtype=torch.int8, device="cuda")]
    scales = [torch.full((1, n), v, device="cuda") for n, v in ((I, 1.71 * 2.0 ** gate), (I, 1.0), (H, 1.19 * 2.0 ** down))]
    layer = i8.I8MoeLayer(*[i8.I8ExpertBank(b, s, k) for b, s, k in zip(banks, scales, (H, H, I))], top_k=1, act=ops.ExpertAct(1, 1.0, 7.0))
    xs = torch.full((T,), 1.37 * 2.0 ** -35, device="cuda")
    out = layer.forward(i8.I8Rows(x, xs, H), randn(g, T, 1))[0]
    h = (x.double() @ w.double()) * xs.double() * scales[0][0, 0].double() / 2  # (the sigmoid is a half to within 2^-80)
    want = (h * I * 127 * scales[2][0, 0].double())[:, None].expand(T, H)
    assert float(want.min()) > 2.0 ** -121 and float(h.min()) > 2.0 ** -126
    # g's rounding, the activation's 10, the hidden scale's (which may be subnormal) and the output's
    slack = I * 127 * 127 * float(scales[2][0, 0]) * 2.0 ** -150
    err = (out.double() - want).abs()
    assert (err <= 1.001 * (13 * U * want + slack)).all(), float((err / want).max() / U)
