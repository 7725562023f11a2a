"""What the products of 8-bit floats keep of codes far apart: results in f16 are those in f32, rounded once; results in bf16 leave out what the
matrix instruction on 8-bit codes cuts, 2^-13 of the largest of 8 neighbouring products for each of the others."""
import pytest
import torch

from coachwhip_amd import f8, ops, piles
from tests.f8_rules import product
from tests.test_f8_dispatch import EXPERTS, INSTANCES
from tests.test_gpu_f8 import gen, rand_bank, rand_matrix, rand_rows, randn, say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
E4M3 = torch.float8_e4m3fn


def far_apart(g, *shape, k, large, small):
    """Codes of which one of 8 neighbours is `large` and seven are `small`, whose products the 8-bit instruction loses whole."""
    q = torch.zeros((*shape, f8.row_bytes(k)), device="cuda")
    q[..., :k] = small
    q[..., :k:8] = large * (2.0 * torch.randint(0, 2, shape, generator=g, device="cuda")[..., None] - 1)
    return q.to(E4M3)


def scales(g, *shape):
    return 2.0 ** -16 * (1 + torch.rand(shape, generator=g, device="cuda"))


def check(y, xq, sx, wq, sw, k, bias):
    """y = 0 + what is lost: the bias takes the sum of the first row away."""
    xv = (xq.double().view(len(xq), -1, 128) * sx.t().double()[..., None]).view(len(xq), -1)
    wv = wq.double() * sw.double().repeat_interleave(128, 0)[:len(wq)].repeat_interleave(128, 1)
    want, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    off = (2 * 128 + sw.shape[1] + 16) * U * size + (7 * 2.0 ** -13 * size if y.dtype == torch.bfloat16 else 0.0)
    want = want + bias.double()
    off = off + U * (want.abs() + bias.double().abs())
    info = torch.finfo(y.dtype)
    assert ((y.double() - want).abs() <= off + info.eps / 2 * (want.abs() + off) + info.smallest_normal * info.eps).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("exact,m,n,k", INSTANCES)
def test_codes_far_apart(exact, m, n, k, dtype):
    if exact != (dtype != torch.bfloat16):
        return
    say(product(exact, m, n, k), m, n, k, dtype)
    g = gen(m + n)
    xq, wq = far_apart(g, m, k=k, large=256.0, small=1.875), far_apart(g, n, k=k, large=256.0, small=3.75)
    sx, sw = scales(g, f8.blocks(k), m), scales(g, f8.blocks(n), f8.blocks(k))
    x, w = f8.F8Rows(xq, sx, k), f8.F8Matrix(wq, sw, k)
    bias = -f8.F8MatMul(w)(f8.F8Rows(xq[:1].contiguous(), sx[:, :1].contiguous(), k))[0]
    check(f8.F8MatMul(w, bias)(x, dtype), xq, sx, wq, sw, k, bias)


@pytest.mark.parametrize("exact,m,n,k", [i for i in INSTANCES if i[0]])
def test_f16_is_f32_rounded(exact, m, n, k):
    say("f16", product(exact, m, n, k), m, n, k)
    g = gen(m + n + k)
    x, w, b = rand_rows(g, m, k), rand_matrix(g, n, k), randn(g, n)
    assert torch.equal(f8.F8MatMul(w, b)(x, torch.float16), f8.F8MatMul(w, b)(x).half())


@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("form,size", [(f, s) for f, sizes in EXPERTS.items() for s in sizes if s[0]])
def test_f16_of_experts_is_f32_rounded(form, size, by_token):
    _, t, e, kp, n, k = size
    say("f16 experts", form, size, by_token)
    g = gen(t + n)
    p = piles.sort_picks(torch.randint(-1, e, (t, kp), generator=g, device="cuda", dtype=torch.int32), e)
    x, product = rand_rows(g, t if by_token else t * kp, k), f8.F8ExpertMatMul(rand_bank(g, e, n, k), randn(g, e, n))
    assert torch.equal(product.forward(x, p, torch.float16, by_token=by_token), product.forward(x, p, by_token=by_token).half())


@pytest.mark.parametrize("t,e,kp,h,i", [(1, 8, 2, 1000, 100), (2, 40, 6, 4000, 1200), (8, 8, 7, 2048, 1000), (700, 16, 4, 513, 300), (700, 4, 2, 384, 1000), (2100, 256, 4, 300, 260)])
def test_f16_of_layers_is_f32_rounded(t, e, kp, h, i):
    say("f16 layer", t, e, kp, h, i)
    g = gen(t + h)
    banks = [rand_bank(g, e, *s) for s in ((i, h), (i, h), (h, i))]
    for b in banks:
        b.scale.mul_(0.3 / b.k ** 0.5)
    act = ops.ExpertAct.clamped_swiglu(1.702, 7.0, *(0.05 * randn(g, e, n) for n in (i, i, h)))
    layer, x, logits = f8.F8MoeLayer(*banks, top_k=kp, act=act), f8.quantize_f8(randn(g, t, h)), randn(g, t, e)
    assert torch.equal(layer.forward(x, logits, torch.float16)[0], layer.forward(x, logits)[0].half())
