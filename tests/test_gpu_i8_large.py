"""The 8-bit integer path where byte offsets pass 32 bits: the far ends of the arrays against the same formulas in 64 bits."""
import pytest
import torch

from coachwhip_amd import i8

from .test_gpu_i8 import Experts, check_codes, check_matmul, gen, rand_rows, randn, say

pytestmark = pytest.mark.gpu


def some(n):
    """The first, middle and last indices below n."""
    return torch.tensor(sorted({0, 1, n // 2, n - 40, n - 2, n - 1}), device="cuda")


def test_rows_past_4_gib():
    say("rows past 4 GiB")
    rows, k = 70_000, 32_768
    x = torch.randn(rows, k, device="cuda", dtype=torch.float16, generator=gen(1))
    r, at = i8.quantize_i8(x), some(70_000)
    check_codes(i8.I8Rows(r.q[at], r.scale[at], k), x[at].double(), 0.0)
    w = 1 + 0.1 * randn(gen(2), k)
    r, total, _ = i8.rmsnorm_i8(x, w, 1e-6, residual=x)
    h = (x[at].float() * 2).half()
    assert torch.equal(total[at], h)
    h = h.double()
    eps = torch.tensor(1e-6, dtype=torch.float32).double().item()
    check_codes(i8.I8Rows(r.q[at], r.scale[at], k), h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w.double(), 1e-13)
    back = r.dequantize(torch.float16)
    assert torch.equal(back[at], i8.I8Rows(r.q[at], r.scale[at], k).dequantize(torch.float16))


@pytest.mark.parametrize("m", [3, 100, 300])
def test_matrix_past_4_gib(m):
    say("matrix past 4 GiB", m)
    n, k = 140_000, 32_768
    g = gen(m)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8), 1 + torch.rand(n, generator=g, device="cuda")
    x, bias, at = rand_rows(g, m, k), randn(g, n), some(n)
    y = i8.I8MatMul(i8.I8Matrix(*w, k), bias)(i8.I8Rows(*x, k))
    check_matmul(x, (w[0][at], w[1][at]), bias[at], torch.float32, y[:, at])


def test_results_past_4_gib():
    say("results past 4 GiB")
    m, n, k = 40_000, 60_000, 128
    g = gen(5)
    x, w, am, an = rand_rows(g, m, k), rand_rows(g, n, k), some(m), some(n)
    y = i8.I8MatMul(i8.I8Matrix(*w, k))(i8.I8Rows(*x, k), torch.bfloat16)
    check_matmul((x[0][am], x[1][am]), (w[0][an], w[1][an]), None, torch.bfloat16, y[am][:, an])


@pytest.mark.parametrize("T", [2, 40])
def test_banks_past_4_gib(T):
    say("banks past 4 GiB", T)
    ex = Experts.__new__(Experts)
    ex.E, ex.H, ex.I, ex.g = 300, 4096, 4096, gen(T)
    ex.w = [(torch.randint(-127, 128, (300, 4096, 4096), generator=ex.g, device="cuda", dtype=torch.int8),
             (0.01 + torch.rand(300, 4096, generator=ex.g, device="cuda")) / (40 * 64), 4096) for _ in range(3)]
    ex.act = i8.ops.ExpertAct.silu()
    x, logits = ex.inputs(T)
    logits[:, 290:] += 4  # the picks among the last experts
    out, ids, w = ex.layer(4).forward(i8.I8Rows(*x, 4096), logits, torch.float32)
    assert (ids >= 256).any()
    ex.check(x, logits, 4, True, out, ids, w)


def test_tokens_past_2_gib():
    say("tokens past 2 GiB")
    T, H = 1_100_000, 2048
    ex = Experts(4, H, 8, "silu", False, 9)
    x, logits = ex.inputs(T)
    out, ids, w = ex.layer(1).forward(i8.I8Rows(*x, H), logits, torch.bfloat16)
    at = torch.cat([some(T), torch.arange(T - 300, T - 100, device="cuda")])
    ex.check((x[0][at], x[1][at]), logits[at], 1, True, out[at], ids[at], w[at])
