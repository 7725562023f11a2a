"""Infinite scales of weights in 8-bit float products of sorted rows, beside those of one matrix."""
import pytest
import torch

from coachwhip_amd import f8, piles
from tests.f8_scales import operands
from tests.test_f8_dispatch import EXPERTS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [100, 260, 600, 1000])
@pytest.mark.parametrize("form,size", [(f, s) for f, sizes in EXPERTS.items() for s in sizes[:2]])
def test_an_infinite_scale_of_the_last_block(form, size, k):
    """Its rows' results are infinite, with the sign of the block's sum, in the experts' kernels as in those of one matrix, whatever the number of k's
    blocks (1, 3, 5, 8) and of those that a kernel takes at a time; the columns beside them keep their bits."""
    exact, t, e, kp, n, _ = size
    print("infinite scale", form, size, k, flush=True)
    ids = torch.randint(0, e, (t, kp), generator=torch.Generator().manual_seed(t), dtype=torch.int32).cuda()
    p = piles.sort_picks(ids, e)
    xq, sx, wq, sw = (a.cuda() for a in operands("tiny", t * kp, n, k, t, e))
    sx.clamp_(max=0.007), sw.clamp_(max=0.007)
    x, dtype = f8.F8Rows(xq, sx, k), torch.float32 if exact else torch.bfloat16
    clean = f8.F8ExpertMatMul(f8.F8ExpertBank(wq, sw.clone(), k)).forward(x, p, dtype)
    sw[:, 1, -1] = float("inf")
    y = f8.F8ExpertMatMul(f8.F8ExpertBank(wq, sw, k)).forward(x, p, dtype)
    last, offsets = 128 * (f8.blocks(k) - 1), p.offsets.tolist()
    for i in range(0, e, max(1, e // 8)):
        at = slice(offsets[i], offsets[i + 1])
        part = xq[at, last:].double() @ wq[i, 128:256, last:].double().t()
        want = torch.where(part == 0, float("nan"), torch.copysign(torch.full_like(part, float("inf")), part))
        assert torch.equal(y[at, 128:256].double().nan_to_num(0.0, 1.0, -1.0), want.nan_to_num(0.0, 1.0, -1.0))
        one = f8.F8MatMul(f8.F8Matrix(wq[i], sw[i], k))(f8.F8Rows(xq[at], sx[:, at].contiguous(), k), dtype)
        assert torch.equal(one[:, 128:256].double().nan_to_num(0.0, 1.0, -1.0), want.nan_to_num(0.0, 1.0, -1.0))
    assert torch.equal(y[:, :128], clean[:, :128]) and torch.equal(y[:, 256:], clean[:, 256:])
