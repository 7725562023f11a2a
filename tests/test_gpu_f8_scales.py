"""8-bit float products whose scales leave f32's range while the results do not, in every kernel (tests/test_f8_scales.py: sums in f32
alone fail on these inputs)."""
import pytest
import torch

from coachwhip_amd import f8, piles
from tests.f8_rules import product
from tests.f8_scales import KINDS, USUAL, operands, result
from tests.test_f8_dispatch import EXPERTS, INSTANCES

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def types_of(exact):
    return [torch.float32, torch.float16] if exact else [torch.bfloat16]


def on_device(*a):
    return [t.cuda() for t in a]


def check(got, want_off):
    want, off = want_off
    assert ((got.double() - want).abs() <= off).all()


def check_matmul(exact, m, n, k, kind, power=62):
    say(product(exact, m, n, k), m, n, k, kind, power)
    xq, sx, wq, sw = on_device(*operands(kind, m, n, k, m + n, power=power))
    bias = None if kind == "under" else torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    for dtype in types_of(exact):
        if dtype in KINDS[kind]:
            check(f8.F8MatMul(f8.F8Matrix(wq[0], sw[0], k), bias)(f8.F8Rows(xq, sx, k), dtype), result(kind, xq, sx, wq[0], sw[0], k, dtype, bias))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("exact,m,n,k", INSTANCES)
def test_products(exact, m, n, k, kind):
    check_matmul(exact, m, n, k, kind)


@pytest.mark.parametrize("power", [USUAL, USUAL + 1, 55, 63])
@pytest.mark.parametrize("exact,m,n,k", [i for i in INSTANCES if i[1] in (16, 120, 500)])
def test_products_of_large_usual_scales(exact, m, n, k, power):
    check_matmul(exact, m, n, k, "cancel", power)


def check_experts(form, size, by_token, kind, power=62):
    exact, t, e, kp, n, k = size
    say("experts", form, size, by_token, kind, power)
    ids = torch.randint(-1, e, (t, kp), generator=torch.Generator().manual_seed(t), dtype=torch.int32).cuda()
    p = piles.sort_picks(ids, e)
    xq, sx, wq, sw = on_device(*operands(kind, t if by_token else t * kp, n, k, t + n, e, power))
    bias = None if kind == "under" else torch.randn(e, n, generator=torch.Generator().manual_seed(n)).cuda()
    offsets = p.offsets.tolist()
    for dtype in types_of(exact):
        if dtype not in KINDS[kind]:
            continue
        y = f8.F8ExpertMatMul(f8.F8ExpertBank(wq, sw, k), bias).forward(f8.F8Rows(xq, sx, k), p, dtype, by_token=by_token)
        assert (y[offsets[e]:] == 0).all()
        for i in range(e):
            rows = torch.arange(offsets[i], offsets[i + 1], device="cuda")
            src = p.order[rows].long() // kp if by_token else rows
            x = xq.view(torch.uint8)[src].view(xq.dtype)
            check(y[rows], result(kind, x, sx[:, src], wq[i], sw[i], k, dtype, None if bias is None else bias[i]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("form,size", [(f, s) for f, sizes in EXPERTS.items() for s in sizes])
def test_experts(form, size, by_token, kind):
    check_experts(form, size, by_token, kind)


@pytest.mark.parametrize("power", [USUAL, USUAL + 1, 63])
@pytest.mark.parametrize("form,size", [(f, s) for f, sizes in EXPERTS.items() for s in sizes[:2]])
def test_experts_of_large_usual_scales(form, size, power):
    check_experts(form, size, True, "cancel", power)
