"""A whole MoE block on 8-bit rows against the same block in 64-bit floats that rounds nothing to codes (the weights are what their
codes stand for). What the roundings may make of an output is estimated as of independent errors, which add in squares: to first
order through the block's slopes, each error as large as this input's own rounding. The host tests show what the comparison
refuses."""
import pytest
import torch


def silu(v):
    return v * torch.sigmoid(v)


def slope(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def code_values(y):
    """What the 8-bit codes of y's rows stand for."""
    step = y.abs().amax(-1, keepdim=True) / 127
    return (y / step).round() * step


def expert(y, wg, wu, wd, scale, rounding):
    """(scale * down(silu(gate y) up y), its slopes to y, the variance that the roundings after y add), y of H values: g
    and u rounded to `rounding` of themselves at most, h to codes."""
    g, u = wg @ y, wu @ y
    h = silu(g) * u
    dg, du = slope(g) * u, silu(g)
    slopes = wd @ (dg[:, None] * wg + du[:, None] * wu)
    var = (h - code_values(h[None])[0]) ** 2 + ((dg * g) ** 2 + (du * u) ** 2) * rounding ** 2 / 3
    return scale * (wd @ h), scale * slopes, scale ** 2 * (wd ** 2 @ var)


def block64(h, norm, router, ids, experts, shared, eps, rounding):
    """((out, its standard error), (shared, its)) of rows h, whose picks are ids. experts: id -> (gate, up, down) in 64 bits; shared:
    the same of one expert, whose g and u are rounded as well. Outputs are rounded to `rounding` of themselves."""
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * norm
    dy = y - code_values(y)
    p = torch.softmax(y @ router.t(), 1).gather(1, ids)
    p = p / p.sum(1, keepdim=True)
    res = []
    for t in range(len(h)):
        parts = [expert(y[t], *experts(int(e)), p[t, j], 0.0) for j, e in enumerate(ids[t])], [expert(y[t], *shared, 1.0, rounding)]
        for which in parts:
            v, s, var = (sum(col) for col in zip(*which))
            res.append((v, torch.sqrt(s ** 2 @ dy[t] ** 2 + var + (rounding * v) ** 2 / 3)))
    stack = lambda k, n: torch.stack([r[n] for r in res[k::2]])
    return (stack(0, 0), stack(0, 1)), (stack(1, 0), stack(1, 1))


def agrees(got, want, err):
    """Errors in units of what is expected of them: normally distributed, nearly, so that none of 50,000 is beyond 7 (once in 10^7
    such sets) and their root mean square is 1; a quarter is left for the second order of the slopes and for few tokens. The
    expected error is small beside the outputs: a comparison that can fail."""
    z = (got.double() - want) / err
    assert err.square().mean().sqrt() <= 0.2 * want.square().mean().sqrt(), "the expected error hides the outputs"
    return bool(z.abs().max() <= 7 and z.square().mean().sqrt() <= 1.25)


# ------------------------------------------------------------------------------ on the host: what the comparison refuses


def host_block(T, seed, E=8, K=3, H=192, I=96):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    x = r(T, H)
    x[:, ::48] *= 4
    w = [[code_values(r(*s) / s[1] ** 0.5) for s in ((I, H), (I, H), (H, I))] for _ in range(E + 1)]
    return x.to(torch.bfloat16).double(), 1 + 0.2 * r(H), r(E, H) / H ** 0.5, w, K


def rounded_block(x, norm, router, w, K, swap=None):
    """The block as the 8-bit path defines it, outputs in bf16; with `swap` one token's first pick goes to that expert."""
    bf = lambda v: v.to(torch.bfloat16).double()
    y = x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-6) * norm
    p = torch.softmax(y @ router.t(), 1)
    ids = p.topk(K, 1)[1]
    p = p.gather(1, ids)
    p = p / p.sum(1, keepdim=True)
    yq = code_values(y)
    out, shared = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(len(x)):
        for j, e in enumerate(ids[t].tolist()):
            wg, wu, wd = w[swap if swap is not None and t == 0 and j == 0 else e]
            h = silu(wg @ yq[t]) * (wu @ yq[t])
            out[t] += p[t, j] * (wd @ code_values(h[None])[0])
        wg, wu, wd = w[-1]
        shared[t] = wd @ code_values((silu(bf(wg @ yq[t])) * bf(wu @ yq[t]))[None])[0]
    return bf(out), bf(shared), ids


@pytest.mark.parametrize("T,seed", [(1, 1), (1, 2), (5, 3), (40, 4)])
def test_the_comparison_on_the_host(T, seed):
    x, norm, router, w, K = host_block(T, seed)
    out, shared, ids = rounded_block(x, norm, router, w, K)
    wants = block64(x, norm, router, ids, lambda e: w[e], w[-1], 1e-6, 2.0 ** -8)
    other = next(e for e in range(8) if e not in ids[0].tolist())
    for got, (want, err), swapped in zip((out, shared), wants, rounded_block(x, norm, router, w, K, other)[:2]):
        assert agrees(got, want, err)
        wrong = [got * 0, -got, got.roll(1, 1), got * 1.5, got + 3 * err]
        if got is out:
            wrong.append(swapped)
        if T > 1:
            wrong.append(got.roll(1, 0))
        assert not any(agrees(v, want, err) for v in wrong)


# ------------------------------------------------------------------------------ the path


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 70])
def test_block_follows_unrounded_floats(T):
    from .test_gpu_i8 import Block, gen, randn, say
    say("block against floats", T)
    b, g, H = Block(), gen(T), 640
    x = randn(g, T, H)
    x[:, ::160] *= 4
    x, r = x.to(torch.bfloat16), randn(g, T, H).to(torch.bfloat16)
    total, out, shared, ids = b(x, r)
    h = (x.float() + r.float()).to(x.dtype)
    assert torch.equal(total, h)
    value = lambda q, s, k: q.double()[:, :k] * s.double()[:, None]
    gu, down = (value(m.w.q, m.w.scale, m.w.k) for m in (b.gu, b.down))
    wants = block64(h.double(), b.norm.double(), b.router.double(), ids.long(), lambda e: [value(q[e], s[e], k) for q, s, k in b.ex.w],
                    (gu[:b.I].contiguous(), gu[b.I:].contiguous(), down), 1e-6, 2.0 ** -8)
    for got, (want, err) in zip((out, shared), wants):
        assert agrees(got, want, err)
        assert not any(agrees(v, want, err) for v in (got * 0, -got, got.roll(1, 1), got + 3 * err))
