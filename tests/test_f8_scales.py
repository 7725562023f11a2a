"""The inputs of tests/test_gpu_f8_scales.py do what they say: summed in f32 alone, without a second way for strange scales, every
output that has two of them is wrong by far more than its tolerance, and the others are right (CPU only)."""
import pytest
import torch

from tests.f8_scales import KINDS, USUAL, blocks, in_f32, operands, result, strange_columns, strange_rows


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 60, 130), (20, 300, 384), (70, 700, 1000)])
def test_sums_in_f32_alone_fail(kind, m, n, k):
    xq, sx, wq, sw = operands(kind, m, n, k, m + n)
    got, both = in_f32(xq, sx, wq[0], sw[0]).double(), strange_rows(m)[:, None] & strange_columns(n).repeat_interleave(128)[:n]
    for dtype in KINDS[kind]:
        want, off = result(kind, xq, sx, wq[0], sw[0], k, dtype)
        assert want.isfinite().all() and (want.abs() < torch.finfo(dtype).max).all()
        bad = ~((got - want).abs() <= 8 * off)
        if kind == "cancel":
            assert bad.all()  # (all scales of two blocks are large)
        else:
            assert bad[both].all() and not bad[~both].any()


@pytest.mark.parametrize("power", [USUAL - 1, USUAL])
def test_usual_scales_need_no_second_way(power):
    xq, sx, wq, sw = operands("cancel", 20, 300, 384, 1, power=power)
    want, off = result("cancel", xq, sx, wq[0], sw[0], 384, torch.float32)
    assert ((in_f32(xq, sx, wq[0], sw[0]).double() - want).abs() <= off).all()


def test_the_largest_sum_of_usual_scales_is_finite():
    assert 448.0 ** 2 * 128 * blocks(32768) * 2.0 ** (2 * USUAL) < torch.finfo(torch.bfloat16).max


def test_experts_beside_the_first_are_strange():
    _, sx, _, sw = operands("zeros", 5, 300, 384, 1, experts=3)
    assert (sw[0] < 1).all() and (sw[1:, :, -1] > 1e15).sum() == 2 * int(strange_columns(300).sum()) and (sx[:-1] < 1).all()
