"""Every kernel of the 8-bit float products, at sizes that leave rows, columns and k odd, and of the layer, at its two forms' borders."""
import pytest
import torch

from coachwhip_amd import f8
from tests.f8_rules import product
from tests.test_f8_dispatch import INSTANCES
from tests.test_gpu_f8 import check_layer, check_product, gen, matrix_values, rand_matrix, rand_rows, randn, say, values

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
