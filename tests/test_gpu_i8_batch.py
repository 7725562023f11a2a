"""A row's product does not depend on the rows beside it: not on their number, which picks the kernel, nor on their scales."""
import pytest
import torch

from coachwhip_amd import i8

from .test_gpu_i8 import DTYPES, gen, rand_rows, randn, say

pytestmark = pytest.mark.gpu

N, K = 4001, 700
BATCHES = [1, 16, 20, 130, 500, 700, 900, 2500]  # rows at a time



@pytest.mark.parametrize("unusual", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_alone_and_together(dtype, unusual):
    say("batches", dtype, unusual)
    g = gen(3)
    (xq, xs), (wq, ws) = rand_rows(g, 5000, K), rand_rows(g, N, K)
    ws = ws / K
    if unusual:  # some rows and channels far from the others, and rows that are not finite
        xs[::3] *= 2.0 ** -70
        xs[5::700] = float("nan")
        xs[7::900] = float("inf")
        xs[9::500] = 0
        ws[::5] *= 2.0 ** 64
        ws[3::50] *= 2.0 ** -80
    for bias in (None, randn(g, N)):
        m = i8.I8MatMul(i8.I8Matrix(wq, ws, K), bias)
        whole = m(i8.I8Rows(xq, xs, K), dtype)
        for size in BATCHES:
            for at in range(0, 5000, max(size, 1250)):
                rows = slice(at, min(at + size, 5000))
                part = m(i8.I8Rows(xq[rows].contiguous(), xs[rows].contiguous(), K), dtype)
                assert torch.equal(part.isnan(), whole[rows].isnan()) and torch.equal(part.nan_to_num(0.0), whole[rows].nan_to_num(0.0)), (size, at)
        narrow = i8.I8MatMul(i8.I8Matrix(wq[:300].contiguous(), ws[:300].contiguous(), K), None if bias is None else bias[:300].contiguous())
        part = narrow(i8.I8Rows(xq[:50].contiguous(), xs[:50].contiguous(), K), dtype)
        assert torch.equal(part.nan_to_num(0.0), whole[:50, :300].nan_to_num(0.0))
