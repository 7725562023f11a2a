"""8-bit float products and piles whose operands or results pass 4 GiB: samples of their rows, the last among them."""
import torch
import pytest

from coachwhip_amd import f8, piles
from tests.test_gpu_f8 import check_product, gen, matrix_values, rand_bank, rand_matrix, say, values

pytestmark = pytest.mark.gpu


def many_rows(n, k, seed):
    """n rows of k codes, the same 4,096 over and over."""
    g = gen(seed)
    part = (torch.randn(4096, k, generator=g, device="cuda") * 100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    q = part.repeat((n + 4095) // 4096, 1)[:n].contiguous().view(torch.float8_e4m3fn)
    return f8.F8Rows(q, 0.001 + 0.01 * torch.rand((f8.blocks(k), n), generator=g, device="cuda"), k)


def some(x, at):
    return values(f8.F8Rows(x.q.view(torch.uint8)[at].view(torch.float8_e4m3fn), x.scale[:, at].contiguous(), x.k))


def test_many_rows_times_a_matrix():
    m, k, n = 140001, 32768, 40
    say("matmul", m, n, k)
    x, w = many_rows(m, k, 1), rand_matrix(gen(2), n, k)
    at = torch.tensor([0, 70000, 131071, 131072, 131073, m - 2, m - 1], device="cuda")
    y = f8.F8MatMul(w)(x, torch.bfloat16)
    check_product(y[at], some(x, at), matrix_values(w.q, w.scale, k), None, torch.bfloat16, k)


def test_many_tokens_times_their_experts():
    t, k, n, e = 140001, 32768, 40, 3
    say("experts", t, n, k)
    x, bank = many_rows(t, k, 3), rand_bank(gen(4), e, n, k)
    ids = (torch.arange(t, device="cuda", dtype=torch.int32) % e)[:, None].contiguous()
    p = piles.sort_picks(ids, e)
    y = f8.F8ExpertMatMul(bank).forward(x, p, torch.bfloat16, by_token=True)
    at = torch.tensor([0, 65535, 131072, 131073, 131074, t - 2, t - 1], device="cuda")
    for i in range(e):
        mine = at[ids[at, 0] == i]
        check_product(y[p.place[mine].long()], some(x, mine), matrix_values(bank.q[i], bank.scale[i], k), None, torch.bfloat16, k)


def test_many_rows_to_the_piles_and_back():
    t, kp, e, h = 70001, 8, 5, 4096  # 4.6 GB of sorted rows
    say("piles", t, kp, h)
    g = gen(5)
    ids = torch.randint(-1, e, (t, kp), generator=g, device="cuda", dtype=torch.int32)
    p = piles.sort_picks(ids, e)
    x = torch.randn(t, h, generator=g, device="cuda").bfloat16()
    rows = piles.to_piles(x, p)
    picks = torch.tensor([0, 1, 131072, t * kp // 2, t * kp - 2, t * kp - 1], device="cuda")
    pos = torch.cat([p.place[picks].long(), torch.tensor([p.offsets[e].item() - 1, p.offsets[e].item(), t * kp - 1], device="cuda")])
    src = p.order[pos].long()
    want = torch.where(((ids.view(-1)[src] >= 0))[:, None], x[src // kp], torch.zeros_like(x[:1]))
    assert torch.equal(rows[pos], want)
    w = torch.rand(t, kp, generator=g, device="cuda")
    tok = torch.tensor([0, 1, t // 2, t - 2, t - 1], device="cuda")
    here = (ids[tok] >= 0).double()
    back = piles.from_piles(rows, w, p)
    want = (w[tok].double() * here).sum(1, keepdim=True) * x[tok].double()
    assert ((back[tok].double() - want).abs() <= (2.0 ** -8 + 9 * 2.0 ** -24) * want.abs() + 1e-30).all()
    drows, dw = piles.from_piles_grad(x, rows, w, p)
    size = x[tok].double().square().sum(1, keepdim=True)
    assert ((dw[tok].double() - here * size).abs() <= (h + 8) * 2.0 ** -24 * size).all()
    pos = p.place.view(t, kp)[tok].long()
    want = (w[tok].double() * here)[..., None] * x[tok].double()[:, None]
    assert ((drows[pos].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -24) * want.abs() + 1e-30).all()
