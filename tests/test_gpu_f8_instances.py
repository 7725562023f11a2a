"""Every kernel of the 8-bit float products, at sizes that leave rows, columns and k odd, and of the layer, at its two forms' borders."""
import pytest
import torch

from coachwhip_amd import f8, piles
from tests.f8_rules import product
from tests.test_f8_dispatch import EXPERTS, INSTANCES
from tests.test_gpu_f8 import check_experts, check_layer, check_product, gen, matrix_values, rand_bank, rand_matrix, rand_rows, randn, say, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exact,m,n,k", INSTANCES)
def test_products(exact, m, n, k):
    say(product(exact, m, n, k), m, n, k)
    g = gen(m + n + k)
    for dtype in ([torch.float32] if exact else [torch.float16, torch.bfloat16]):
        x, w, b = rand_rows(g, m, k), rand_matrix(g, n, k), randn(g, n)
        check_product(f8.F8MatMul(w, b)(x, dtype), values(x), matrix_values(w.q, w.scale, k), b, dtype, k)


# hidden and inter of every number of steps that the kernels for a few tokens are built for; experts beyond a lane's 4 and 8 logits
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("e,kp,h,i", [(8, 1, 1000, 100), (8, 2, 1100, 500), (300, 4, 2100, 1000), (600, 5, 4000, 1200), (1024, 6, 300, 2000), (40, 32, 500, 500), (8, 7, 4096, 2300)])
def test_layers_of_a_few_tokens(e, kp, h, i, dtype):
    say("few tokens", e, kp, h, i, dtype)
    check_layer(2, e, kp, h, i, dtype, True)


@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("form,size", [(f, s) for f, sizes in EXPERTS.items() for s in sizes])
def test_experts(form, size, by_token):
    exact, t, e, kp, n, k = size
    say("experts", form, size, by_token)
    ids = torch.randint(-1, e, (t, kp), generator=gen(t), device="cuda", dtype=torch.int32)
    for dtype in ([torch.float32] if exact else [torch.float16, torch.bfloat16]):
        check_experts(t, e, kp, n, k, dtype, True, by_token, ids)


@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("form,size", [(f, sizes[1]) for f, sizes in EXPERTS.items()])
def test_experts_scales_of_any_size(form, size, by_token):
    """Scales of one group of k whose product leaves f32's range in two blocks of all experts' outputs but the first's, while the results do not."""
    _, t, e, kp, n, k = size
    say("experts with scales of any size", form, size, by_token)
    g = gen(t + n)
    p = piles.sort_picks(torch.randint(0, e, (t, kp), generator=g, device="cuda", dtype=torch.int32), e)
    bank, x, b = rand_bank(g, e, n, k), rand_rows(g, t if by_token else t * kp, k), randn(g, e, n)
    x.scale[1] *= 2.0 ** 100
    bank.scale[1:, 1:, 1] *= 2.0 ** -100
    y = f8.F8ExpertMatMul(bank, b).forward(x, p, torch.float32, by_token=by_token)
    xv, offsets = values(x), p.offsets.tolist()
    for i in range(e):
        at = slice(offsets[i], offsets[i + 1])
        rows = xv[p.order[at].long() // kp] if by_token else xv[at]
        for c in range(0, n, 128):
            check_product(y[at, c:c + 128], rows, matrix_values(bank.q[i], bank.scale[i], k)[c:c + 128], b[i, c:c + 128], torch.float32, k)
