"""Piles of the widest rows that the calls take, 2^31 - 1 values: places near the end of what 32 bits count."""
import torch
import pytest

from coachwhip_amd import piles

pytestmark = pytest.mark.gpu

H = 2 ** 31 - 1
AT = [0, 511, 512, 2 ** 30, H - 1024, H - 513, H - 512, H - 511, H - 9, H - 8, H - 7, H - 1]


def test_the_widest_rows():
    print("piles of rows of", H, flush=True)
    p = piles.sort_picks(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), 1)
    at = torch.tensor(AT, device="cuda")
    x = torch.zeros(1, H, dtype=torch.bfloat16, device="cuda")
    x[0, at] = torch.arange(1, len(AT) + 1, device="cuda").bfloat16()
    rows = piles.to_piles(x, p)
    assert torch.equal(rows[0, at], x[0, at]) and torch.count_nonzero(rows) == len(AT)
    w = torch.full((1, 1), 3.0, device="cuda")
    back = piles.from_piles(rows, w, p)
    assert torch.equal(back[0, at], 3 * x[0, at]) and torch.count_nonzero(back) == len(AT)
    del back
    drows, dw = piles.from_piles_grad(x, rows, w, p)
    assert torch.equal(drows[0, at], 3 * x[0, at]) and torch.count_nonzero(drows) == len(AT)
    assert dw.item() == sum(i * i for i in range(1, len(AT) + 1))
