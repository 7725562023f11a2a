"""The activation of the 8-bit integer path value by value: in rows of one value the scale is |h| / 127, so that f32's last
bits show, as no code of a row shows them."""
import pytest
import torch

from coachwhip_amd import i8, ops

from .test_gpu_i8 import U, gen, glu64, randn, say

pytestmark = pytest.mark.gpu

# In half steps of f32: 2^x is within a step (2), its sum with 1 (1), 1 / x within a step (2), the correction for the exponent's
# rounding (1; its own error is below 2^-35), the products and u + 1 (3), the scale (1). What the exponent is rounded by is
# corrected: the bound does not grow with |g|.
HALF_STEPS = 10.01


def acts():
    f32 = lambda v: torch.tensor(v, dtype=torch.float32).item()  # the constants as the call takes them
    return {"silu": ops.ExpertAct.silu(), "clamped": ops.ExpertAct(1, f32(1.702), 7.0), "steep": ops.ExpertAct(1, f32(7.31), f32(11.3))}


def gates(act, n):
    """From where 2^x is about 2^-115 to where it is about 2^115."""
    a = act.alpha if act.kind else 1.0
    return torch.linspace(-80 / a, 80 / a, n, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", sorted(acts()))
def test_swiglu_keeps_f32_accuracy(name, dtype):
    say("swiglu value by value", name, dtype)
    act = acts()[name]
    g = gates(act, 50_001).to(dtype)[:, None]
    u = (3 * randn(gen(1), 50_001, 1)).to(dtype)
    r = i8.swiglu_i8(g, u, act)
    want = glu64(g.double(), u.double(), act).abs()
    err = (r.scale.double()[:, None] * 127 - want).abs()
    assert (err <= HALF_STEPS * U * want + 127 * 2.0 ** -149).all(), float((err / want.clamp(min=1e-30)).max() / U)


def test_swiglu_at_the_ends_of_f32():
    big = torch.finfo(torch.float32).max
    g = torch.tensor([big, -big, 3e38, -3e38, 2.4e38, -2.4e38, 1e30, -1e30, 200.0, -200.0, 0.0, float("nan"), float("inf")], device="cuda")[:, None]
    u = torch.full_like(g, 0.5)
    got = i8.swiglu_i8(g, u).scale * 127
    want = torch.where(g[:, 0] > 0, g[:, 0] / 2, 0.0).double()
    assert torch.isnan(got[11:]).all()
    assert ((got[:11].double() - want[:11]).abs() <= HALF_STEPS * U * want[:11] + 2.0 ** -126).all()
    act = acts()["clamped"]
    got = i8.swiglu_i8(g, u, act).scale * 127
    top = glu64(torch.tensor(7.0, dtype=torch.float64), torch.tensor(0.5, dtype=torch.float64), act)
    want = torch.where(g[:, 0] > 0, float(top), 0.0).double()
    assert torch.isnan(got[11]) and ((got[:11].double() - want[:11]).abs() <= HALF_STEPS * U * want[:11] + 2.0 ** -126).all()


@pytest.mark.parametrize("T", [5, 700, 1030])  # (in two launches, and grouped)
@pytest.mark.parametrize("name", ["silu", "clamped"])
def test_layer_keeps_f32_accuracy(name, T):
    """One expert of one hidden value: g and u are exact (scales of few bits), the hidden row's code is 127 or -127, and
    each output h * 127 / 127 * 127: the scale's rounding and the output's beside the activation's."""
    say("layer value by value", name, T)
    act, H, gq = acts()[name], 128, gen(T)
    q = lambda *shape: torch.zeros(shape, dtype=torch.int8, device="cuda")
    w = [q(1, 1, 128), q(1, 1, 128), q(1, H, 128)]
    w[0][0, 0, 0] = w[1][0, 0, 1] = 1
    w[2][0, :, 0] = 127
    scales = [0.375, 0.0625, 1.0]  # (g up to 47.6: 1 / (1 + 2^-x) stays a normal number)
    layer = i8.I8MoeLayer(*[i8.I8ExpertBank(v, torch.full(v.shape[:2], s, device="cuda"), k) for v, s, k in zip(w, scales, (H, H, 1))], top_k=1, act=act)
    x = q(T, H)
    x[:, :2] = torch.randint(-127, 128, (T, 2), generator=gq, device="cuda")
    out = layer.forward(i8.I8Rows(x, torch.ones(T, device="cuda"), H), randn(gq, T, 1))[0]
    h = glu64(x[:, 0].double() * 0.375, x[:, 1].double() * 0.0625, act)
    want = (h * 127)[:, None].expand(T, H)
    err = (out.double() - want).abs()
    assert (err <= (HALF_STEPS + 1) * U * want.abs() + 127 * 127 * 2.0 ** -149).all(), float((err / want.abs().clamp(min=1e-30)).max() / U)
