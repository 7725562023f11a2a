"""Layers of 8-bit float experts in every kernel that they can take (tests/test_f8_layer_forms.py): against 64 bits, with scales whose
products leave f32's range, and a token that is not finite beside others."""
import pytest
import torch

from coachwhip_amd import f8
from tests.f8_layer_oracle import layer_64
from tests.f8_layer_rules import FEW, GROUPED
from tests.test_gpu_f8 import check_layer, gen, rand_bank, randn, say

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZES = [("few", s) for s in FEW] + [(form, s) for form, sizes in GROUPED.items() for s in sizes]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("form,size", SIZES)
def test_layers_match_64_bits(form, size, act, dtype):
    say("layer", form, size, act, dtype)
    check_layer(*size, dtype, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form,size", [x for x in SIZES if x[1][0] > 1])
def test_a_token_that_is_not_finite_stays_alone(form, size, dtype):
    say("not finite", form, size, dtype)
    layer, x, logits, out = check_layer(*size, dtype, True)
    t, bad = size[0], size[0] // 2
    x.scale[-1, bad] = float("nan")
    got, _, _ = layer.forward(x, logits, dtype)
    keep = torch.arange(t, device="cuda") != bad
    assert got[bad].isnan().all() and torch.equal(got[keep], out[keep])


def pieces(t, e, kp, h, i):
    g = gen(t + h)
    banks = [rand_bank(g, e, *s) for s in ((i, h), (i, h), (h, i))]
    for b in banks:
        b.scale.mul_(0.3 / b.k ** 0.5)
    return banks, f8.quantize_f8(randn(g, t, h)), randn(g, t, e)


def check(banks, x, logits, top_k, dtype):
    got, ids, w = f8.F8MoeLayer(*banks, top_k=top_k).forward(x, logits, dtype)
    want, off = layer_64(banks, x, ids, w, dtype)
    assert want.isfinite().all() and ((got.double() - want).abs() <= off).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form,size", SIZES)
def test_strange_scales_of_gate_and_up(form, size, dtype):
    """The last block of the hidden size has zero codes in x, and scales whose product overflows: no infinity times zero."""
    say("strange gate and up", form, size, dtype)
    banks, x, logits = pieces(*size)
    last = 128 * (f8.blocks(size[3]) - 1)
    x.q.view(torch.uint8)[:, last:] = 0
    check(banks, x, logits, size[2], dtype)
    x.scale[-1] = 2.0 ** 70
    for b in banks[:2]:
        b.scale[:, ::2, -1] = 2.0 ** 70
    check(banks, x, logits, size[2], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form,size", [x for x in SIZES if x[1][4] > 128])
def test_strange_scales_of_down(form, size, dtype):
    """The first block of the hidden rows is large (2^20 times the others), and down has zero codes for it and a scale whose product with its rows'
    overflows."""
    say("strange down", form, size, dtype)
    banks, x, logits = pieces(*size)
    banks[1].scale[:, 0] *= 2.0 ** 20
    banks[2].q.view(torch.uint8)[:, :, :128] = 0
    check(banks, x, logits, size[2], dtype)
    banks[2].scale[:, ::2, 0] = 2.0 ** 125
    check(banks, x, logits, size[2], dtype)
