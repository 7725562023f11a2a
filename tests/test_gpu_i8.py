"""The 8-bit integer path against the same formulas in 64 bits.

Integer sums are exact, so a product is off by its scalings alone; a code is the nearest integer, so it may differ
from the oracle's only where the value lies as near to the border between two codes as its own error."""
import itertools

import pytest
import torch

import coachwhip_amd as cw
from coachwhip_amd import formats as F
from coachwhip_amd import i8, ops, synth

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24  # half a step of f32


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def say(*a):
    print(*a, flush=True)


def codes_of(rows):
    assert rows.q.shape[1] == i8.row_bytes(rows.k) and not rows.q[:, rows.k:].any()
    return rows.q[:, :rows.k].double()


def check_codes(rows, y, rel):
    """rows against y in 64 bits, whose f32 values are off by rel of themselves at most: scales by rel and their rounding, codes
    by 127 * 2 rel (their value's error and that of the largest) before they are rounded."""
    a = y.abs().amax(1)
    assert ((rows.scale.double() - a / 127).abs() <= (rel + U) * a / 127 + 2.0 ** -150).all()
    v = y * (127 / a.clamp(min=1e-300))[:, None]
    got, near = codes_of(rows), 254 * rel + 1e-9
    assert ((got - v).abs() <= 0.5 + near).all()


def make_rows(g, n, k, loud=4):
    x = randn(g, n, k)
    x[:, :: max(1, k // loud)] *= 9
    return x


def rand_rows(g, n, k):
    q = torch.zeros((n, i8.row_bytes(k)), dtype=torch.int8, device="cuda")
    q[:, :k] = torch.randint(-127, 128, (n, k), generator=g, device="cuda")
    return q, 0.01 + torch.rand(n, generator=g, device="cuda")


# ------------------------------------------------------------------------------ rows to codes

ROW_SHAPES = [(1, 1), (3, 7), (1, 128), (2, 129), (5, 512), (4, 1000), (1, 2048), (7, 2880), (3, 4097), (2, 8192), (2, 9001), (1, 32768), (1030, 66), (2053, 2881)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", ROW_SHAPES)
def test_quantize_matches_64_bits(rows, k, dtype):
    say("quantize", rows, k, dtype)
    x = make_rows(gen(k), rows, k).to(dtype)
    r = i8.quantize_i8(x)
    check_codes(r, x.double(), 0.0)
    for out in DTYPES:
        want = codes_of(r) * r.scale.double()[:, None]
        assert ((r.dequantize(out).double() - want).abs() <= half(out) * want.abs() + U * want.abs() + torch.finfo(out).tiny).all()


def test_quantize_of_strided_and_unaligned_rows():
    x = make_rows(gen(1), 9, 700).to(torch.float16)
    for part in (x[:, 3:404], x[1::2, 1:], x[:, :1], x[4:5, 5:]):
        r, want = i8.quantize_i8(part), i8.quantize_i8(part.contiguous())
        assert torch.equal(r.q, want.q) and torch.equal(r.scale, want.scale)


def test_rows_of_zeros_tiny_huge_and_not_finite_values():
    x = make_rows(gen(2), 8, 300)
    x[1] = 0
    x[2] *= 1e-40  # subnormal
    x[3] *= 1e37
    x[4, 299] = float("nan")
    x[5, 0] = float("inf")
    x[6, 17] = -float("inf")
    r = i8.quantize_i8(x)
    assert r.scale[1] == 0 and not r.q[1].any()
    fine = [0, 2, 3, 7]
    v = x[fine].double()
    assert ((codes_of(r)[fine] - v * 127 / v.abs().amax(1, keepdim=True)).abs() <= 0.5 + 1e-9).all()
    assert torch.isnan(r.scale[4:7]).all() and not r.q[4:7].any()
    assert torch.isnan(r.dequantize()[4:7]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,k", ROW_SHAPES)
def test_rmsnorm_matches_64_bits(rows, k, residual, dtype):
    say("rmsnorm", rows, k, residual, dtype)
    g = gen(100 + k)
    x = make_rows(g, rows, k).to(dtype)
    r = (2 * randn(g, rows, k)).to(dtype) if residual else None
    w = 1 + 0.3 * randn(g, k)
    q, total, y = i8.rmsnorm_i8(x, w, 1e-5, residual=r, keep_y=True)
    h = x
    if residual:
        h = (x.float() + r.float()).to(dtype)
        assert torch.equal(total, h)
    else:
        assert total is None
    eps = torch.tensor(1e-5, dtype=torch.float32).double().item()  # the f32 that the call takes
    want = h.double() / torch.sqrt(h.double().square().mean(1, keepdim=True) + eps) * w.double()
    assert ((y.double() - want).abs() <= U * (1 + 1e-6) * want.abs() + 2.0 ** -150).all()
    check_codes(q, want, 1e-13)
    q2, _, none = i8.rmsnorm_i8(x, w, 1e-5, residual=r)
    assert none is None and torch.equal(q2.q, q.q) and torch.equal(q2.scale, q.scale)


def test_rmsnorm_sum_in_place_and_of_strided_rows():
    g = gen(5)
    big, res, w = make_rows(g, 6, 900).to(torch.bfloat16), randn(g, 6, 900).to(torch.bfloat16), randn(g, 300)
    x, r = big[:, 301:601], res[:, 1:301]
    q, total, _ = i8.rmsnorm_i8(x, w, 1e-6, residual=r)
    want = i8.rmsnorm_i8(x.contiguous(), w, 1e-6, residual=r.contiguous())
    assert torch.equal(total, want[1]) and torch.equal(q.q, want[0].q)
    # the C call may write the sum over the residual
    xc, rc = x.contiguous(), r.contiguous()
    ws = i8.I8Rows(torch.empty_like(q.q), torch.empty_like(q.scale), 300)
    rc_status = cw.lib().cw_rmsnorm_i8(F.BF16, ops._p(xc), 300, ops._p(rc), 300, ops._p(w), 1e-6, 6, 300, ops._p(rc), None, ops._p(ws.q),
                                       ops._p(ws.scale), ops._stream())
    assert rc_status == 0 and torch.equal(rc, total) and torch.equal(ws.q, q.q)


def test_rmsnorm_rows_not_finite_stay_alone():
    g = gen(6)
    x, w = make_rows(g, 4, 513), 1 + 0.1 * randn(g, 513)
    clean, _, _ = i8.rmsnorm_i8(x, w, 1e-6)
    x[1, 3], x[2, 512] = float("inf"), float("nan")
    q, _, _ = i8.rmsnorm_i8(x, w, 1e-6)
    assert torch.isnan(q.scale[1:3]).all() and not q.q[1:3].any()
    assert torch.equal(q.q[0::3], clean.q[0::3]) and torch.equal(q.scale[0::3], clean.scale[0::3])
    zero, _, _ = i8.rmsnorm_i8(torch.zeros(2, 100, device="cuda"), w[:100].contiguous(), 1e-6)
    assert not zero.scale.any() and not zero.q.any()


# h in f32: 2^x within an ulp (2 U) of its argument's value, whose own rounding and that of the constant in it are 2 U of at most
# 8 * 1.702 (as a power of e); 1 / x within an ulp; the two sums and the products a U each
GLU_REL = (2 + 2 * 8 * 1.702 + 2 + 6) * U


def glu64(g, u, act):
    if act.kind == 0:
        return g * torch.sigmoid(g) * u
    g, u = g.clamp(max=act.limit), u.clamp(-act.limit, act.limit)
    return (u + 1) * g * torch.sigmoid(act.alpha * g)


ACTS = {"silu": ops.ExpertAct.silu(), "clamped": ops.ExpertAct.clamped_swiglu(1.702, 7.0, None, None, None)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("rows,k", ROW_SHAPES)
def test_swiglu_matches_64_bits(rows, k, act, dtype):
    say("swiglu", rows, k, act, dtype)
    gu = (2 * randn(gen(200 + k), rows, 2 * k)).clamp(-8, 8).to(dtype)
    r = i8.swiglu_i8(gu[:, :k], gu[:, k:], ACTS[act])
    a = ops.ExpertAct(1, torch.tensor(1.702).item(), 7.0) if act == "clamped" else ACTS[act]  # alpha as f32
    a.alpha = torch.tensor(a.alpha, dtype=torch.float32).item()
    check_codes(r, glu64(gu[:, :k].double(), gu[:, k:].double(), a), GLU_REL)


# ------------------------------------------------------------------------------ products


def check_matmul(x, w, bias, dtype, y):
    """The product p is off by three roundings of f32 (the sum's conversion, the scales' product, the last one), y by its own."""
    p = (x[0].double() @ w[0].double().t()) * x[1].double()[:, None] * w[1].double()
    want = p if bias is None else p + bias.double()
    assert y.dtype == dtype and y.shape == want.shape
    err = (y.double() - want).abs()
    assert (err <= 1.001 * (2 * U * p.abs() + (U + half(dtype)) * want.abs()) + torch.finfo(dtype).tiny).all(), float(err.max())


MM_SHAPES = [(1, 1, 1), (1, 2048, 2048), (2, 17, 100), (1, 513, 4097), (3, 4001, 2880), (15, 64, 128), (16, 4096, 4096), (17, 70, 640), (33, 1000, 257),
             (77, 4001, 2880), (64, 512, 8192), (100, 33, 32768), (128, 256, 384), (129, 255, 896), (130, 2048, 200), (200, 1024, 1024), (300, 777, 1536),
             (513, 513, 513), (1025, 300, 128), (700, 4096, 640),
             # a step or a few in a ring of eight, tiles of 64 x 128, of 128 x 128, of 256 x 256
             (200, 300, 64), (200, 300, 384), (90, 500, 1025), (20, 9000, 2000), (512, 4001, 1500), (400, 4096, 300), (900, 3000, 2500), (3600, 4500, 128),
             (8200, 8200, 100), (4096, 4000, 512), (5000, 3001, 897), (2500, 6001, 300), (5000, 4000, 2000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", MM_SHAPES)
def test_matmul_is_exact_but_for_its_scales(m, n, k, dtype):
    say("matmul", m, n, k, dtype)
    g = gen(m + n + k)
    x, w = rand_rows(g, m, k), rand_rows(g, n, k)
    w[1].mul_(1.0 / k)  # (f16: results within its range)
    for bias in (None, randn(g, n)):
        y = i8.I8MatMul(i8.I8Matrix(*w, k), bias)(i8.I8Rows(*x, k), dtype)
        check_matmul(x, w, bias, dtype, y)


def test_matmul_at_the_largest_sums():
    k = 32768
    for sx, sw in itertools.product((-128, 127), (-128, 127)):
        x = torch.full((2, k), sx, dtype=torch.int8, device="cuda")
        w = torch.full((3, k), sw, dtype=torch.int8, device="cuda")
        one = torch.ones(3, device="cuda")
        y = i8.I8MatMul(i8.I8Matrix(w, one, k))(i8.I8Rows(x, one[:2].clone(), k))
        assert (y.double() == float(torch.tensor(float(sx * sw * k), dtype=torch.float32))).all()


def test_matmul_writes_its_rows_alone():
    """Rows of y wider apart than n: what lies between them, and behind the last, stays."""
    g = gen(9)
    for m, n in ((1, 5), (7, 33), (40, 100), (150, 131)):
        x, w = rand_rows(g, m, 300), rand_rows(g, n, 300)
        y = torch.full((m + 1, n + 6), 7.0, device="cuda")
        assert cw.lib().cw_i8_matmul(ops._p(w[0]), ops._p(w[1]), n, 300, ops._p(x[0]), ops._p(x[1]), m, None, F.F32, ops._p(y), n + 6,
                                     ops._stream()) == 0
        check_matmul(x, w, None, torch.float32, y[:m, :n])
        assert (y[:, n:] == 7).all() and (y[m] == 7).all()


def test_matmul_of_a_row_that_is_not_finite():
    g = gen(10)
    for m in (2, 40, 200):
        x, w = rand_rows(g, m, 256), rand_rows(g, 96, 256)
        clean = i8.I8MatMul(i8.I8Matrix(*w, 256))(i8.I8Rows(*x, 256))
        x[1][1], x[0][1] = float("nan"), 0
        y = i8.I8MatMul(i8.I8Matrix(*w, 256))(i8.I8Rows(*x, 256))
        assert torch.isnan(y[1]).all() and torch.equal(y[0], clean[0]) and torch.equal(y[2:], clean[2:])


def test_weights_from_gguf():
    rng = __import__("numpy").random.default_rng(3)
    q = ops.QTensor.from_blocks(synth.random_blocks(F.Q8_0, 96 * 320, rng), F.Q8_0, (96, 320))
    check_codes(i8.I8Rows(*(lambda m: (m.q, m.scale, m.k))(i8.I8Matrix.from_qtensor(q))), q.dequantize().double(), 0.0)
    bank = ops.ExpertBank.from_blocks(synth.random_blocks(F.Q4_K, 3 * 40 * 512, rng), F.Q4_K, 40, 512, 3)
    b = i8.I8ExpertBank.from_bank(bank)
    w = ops.dequantize(F.Q4_K, bank.data, 3 * 40 * 512).view(3 * 40, 512)
    assert b.q.shape == (3, 40, 512)
    check_codes(i8.I8Rows(b.q.view(120, 512), b.scale.view(120), 512), w.double(), 0.0)
    f = i8.I8ExpertBank.from_float(w.view(3, 40, 512))
    assert torch.equal(f.q, b.q) and torch.equal(f.scale, b.scale)


# ------------------------------------------------------------------------------ the layer


class Experts:
    def __init__(self, E, H, I, act, bias, seed):
        g = gen(seed)
        self.E, self.H, self.I = E, H, I
        self.w = []
        for n, k in ((I, H), (I, H), (H, I)):
            q, s = rand_rows(g, E * n, k)
            self.w.append((q.view(E, n, -1), (s / (40 * k ** 0.5)).view(E, n), k))
        b = [0.3 * randn(g, E, n) for n in (I, I, H)] if bias else [None] * 3
        self.act = ops.ExpertAct(0 if act == "silu" else 1, 1.702, 7.0, *b)
        self.g = g

    def layer(self, K, norm=True):
        return i8.I8MoeLayer(*[i8.I8ExpertBank(*w) for w in self.w], top_k=K, norm_topk_prob=norm, act=self.act)

    def inputs(self, T):
        return rand_rows(self.g, T, self.H), randn(self.g, T, self.E)

    def check(self, x, logits, K, norm, out, ids, w):
        """Gate and up are off by 3 U each and their sum's rounding, h by that and GLU_REL; a code of h that lies that near to a
        border may be its neighbour; the sums of at most 16 terms a lane, 6 levels and 32 picks are within 128 U of the terms'
        magnitudes, the weights within `weight`."""
        order = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :K]
        assert torch.equal(ids.long(), order)
        p = torch.softmax(logits.double(), 1).gather(1, order)
        p = p / p.sum(1, keepdim=True) if norm else p
        weight = (64 + float(logits.max() - logits.min())) * U  # an exp of a rounded difference, a sum, a division
        assert ((w.double() - p).abs() <= weight * p).all()
        xv = x[0].double()[:, :self.H] * x[1].double()[:, None]
        T = xv.shape[0]
        want, slack = torch.zeros(T, self.H, dtype=torch.float64, device="cuda"), torch.zeros(T, self.H, dtype=torch.float64, device="cuda")
        act = ops.ExpertAct(self.act.kind, torch.tensor(self.act.alpha, dtype=torch.float32).item(), self.act.limit)
        bias = [self.act.gate_b, self.act.up_b, self.act.down_b]
        for e in torch.unique(order).tolist():
            t, j = torch.nonzero(order == e, as_tuple=True)
            m = [q[e].double()[:, :k] * s[e].double()[:, None] for q, s, k in self.w]
            b = [0.0 if v is None else v[e].double() for v in bias]
            pg, pu = xv[t] @ m[0].t(), xv[t] @ m[1].t()
            g, u = pg + b[0], pu + b[1]
            h = glu64(g, u, act)
            # d h: the factors' slopes (|silu'| <= 1.1, of the clamped form 1.1 as well) times their errors, and the activation's own
            dg, du = 4 * U * (pg.abs() + g.abs()), 4 * U * (pu.abs() + u.abs())
            gate = (g * torch.sigmoid(act.alpha * g)).abs() if act.kind else (g * torch.sigmoid(g)).abs()
            rel = GLU_REL + (act.alpha if act.kind else 1) * g.abs() * 2 * U  # (of arguments past 8 * 1.702)
            dh = 1.2 * dg * (u.abs() + act.kind) + du * gate + rel * h.abs()
            a = h.abs().amax(1, keepdim=True)
            da = dh.amax(1, keepdim=True)
            v = h * 127 / a
            near = 127 * (dh / a + h.abs() * da / a ** 2) * 1.01
            q = v.round()
            flips = ((v - q).abs() >= 0.5 - near).double() * (1 + near)
            step = a / 127
            want.index_add_(0, t, p[t, j][:, None] * ((q * step) @ m[2].t() + b[2]))
            mag = (q.abs() * step) @ m[2].abs().t() + (b[2].abs() if bias[2] is not None else 0.0)
            slack.index_add_(0, t, p[t, j][:, None] * ((flips * step) @ m[2].abs().t() + (128 * U + weight + da / a) * mag))
        err = (out.double() - want).abs()
        bound = slack + half(out.dtype) * want.abs() + torch.finfo(out.dtype).tiny
        assert (err <= bound).all(), (float(err.max()), float((err / bound).max()))


LAYERS = [  # E, K, H, I, activation, biases
    (8, 2, 100, 36, "silu", False), (5, 5, 130, 129, "clamped", True), (64, 8, 2048, 512, "silu", False), (16, 4, 2880, 700, "clamped", True),
    (300, 10, 256, 128, "silu", True), (1024, 32, 128, 64, "silu", False), (3, 1, 1000, 4096, "silu", False), (4, 2, 4224, 300, "clamped", False),
    (1, 1, 16, 8, "silu", False), (600, 3, 640, 1, "silu", False)]


@pytest.mark.parametrize("T", [1, 3, 8, 9, 40, 300])
@pytest.mark.parametrize("E,K,H,I,act,bias", LAYERS)
def test_layer_matches_64_bits(E, K, H, I, act, bias, T):
    say("layer", E, K, H, I, act, bias, T)
    ex = Experts(E, H, I, act, bias, E + H + I)
    x, logits = ex.inputs(T)
    norm = (T + K) % 3 != 0
    layer = ex.layer(K, norm)
    for dtype in DTYPES if T in (3, 40) else [torch.bfloat16]:
        out, ids, w = layer.forward(i8.I8Rows(*x, H), logits, dtype)
        assert out.dtype == dtype
        ex.check(x, logits, K, norm, out, ids, w)


@pytest.mark.parametrize("T", [129, 600, 1100])
def test_layer_with_every_token_on_one_expert(T):
    ex = Experts(6, 256, 200, "silu", False, 1)
    x, logits = ex.inputs(T)
    logits[:, 4] += 50
    out, ids, w = ex.layer(2).forward(i8.I8Rows(*x, 256), logits, torch.float32)
    assert (ids[:, 0] == 4).all()
    ex.check(x, logits, 2, True, out, ids, w)


@pytest.mark.parametrize("T", [2, 30, 1030])  # (the last grouped)
def test_layer_rows_not_finite_or_zero_stay_alone(T):
    ex = Experts(8, 256, 96, "clamped", True, 2)
    x, logits = ex.inputs(T)
    layer = ex.layer(2)
    clean = layer.forward(i8.I8Rows(*x, 256), logits)[0]
    x[0][1], x[1][1] = 0, float("nan")
    out = layer.forward(i8.I8Rows(*x, 256), logits)[0]
    assert torch.isnan(out[1]).all() and torch.equal(out[0], clean[0]) and torch.equal(out[2:], clean[2:])
    x[1][1] = 0
    out, ids, w = layer.forward(i8.I8Rows(*x, 256), logits)
    ex.check(x, logits, 2, True, out, ids, w)


@pytest.mark.parametrize("T", [5, 1030])  # (in two launches, and grouped)
def test_layer_logits_not_finite_stay_alone(T):
    """The routing is ``ops.route``'s, whatever the logits: picks are experts that exist, each once; a row with a NaN or
    +inf among its logits, or with -inf alone, has NaN results, -inf beside enough finite logits masks an expert, and so does
    a NaN with its sign set, which that order puts below every other value (renormalised weights sum the picks alone)."""
    ex = Experts(70, 256, 96, "clamped", True, 3)
    x, logits = ex.inputs(T)
    layer = ex.layer(4)
    clean = layer.forward(i8.I8Rows(*x, 256), logits)
    bad = logits.clone()
    bad[0, 69] = float("nan")
    bad[1, ::2] = torch.tensor([-1], dtype=torch.int32, device="cuda").view(torch.float32)  # a negative NaN, all bits set
    bad[2] = -float("inf")
    bad[3, 7] = float("inf")
    bad[4, 4:] = -float("inf")
    out, ids, w = layer.forward(i8.I8Rows(*x, 256), bad)
    assert ((0 <= ids) & (ids < 70)).all() and all(len(set(row)) == 4 for row in ids.tolist())
    want_ids, want_w = ops.route(bad, 4, True)
    assert torch.equal(ids, want_ids.to(ids.dtype)) and torch.allclose(w, want_w, rtol=0, atol=0, equal_nan=True)
    assert torch.isnan(out[[0, 2, 3]]).all() and torch.isfinite(out[1]).all() and (ids[1] % 2 == 1).all()
    assert sorted(ids[4].tolist()) == [0, 1, 2, 3] and torch.isfinite(out[4]).all()
    for a, b in zip((out, ids, w), clean):
        assert torch.equal(a[5:], b[5:])


@pytest.mark.parametrize("T", [1, 8, 50])
def test_layer_repeats_its_bits_on_any_workspace(T):
    ex = Experts(16, 512, 256, "silu", False, 3)
    x, logits = ex.inputs(T)
    layer = ex.layer(4)
    first = layer.forward(i8.I8Rows(*x, 512), logits)
    import ctypes
    d = ctypes.byref(layer.desc)
    need = cw.lib().cw_i8_moe_workspace_size(d, T)
    for fill in (0, 0xFF, 0x5A):
        ws = torch.full((need + 256,), fill, dtype=torch.uint8, device="cuda")
        out = torch.empty(T, 512, device="cuda")
        assert cw.lib().cw_i8_moe_layer(d, ops._p(x[0]), ops._p(x[1]), ops._p(logits), T, F.F32, ops._p(out), None, None, ops._p(ws), need,
                                        ops._stream()) == 0
        assert torch.equal(out, first[0]) and (ws[need:] == fill).all()


# ------------------------------------------------------------------------------ together, in graphs and on streams


class Block:
    """A MoE block: norm, router, experts, and a shared expert of three products."""

    def __init__(self, E=16, K=4, H=640, I=320):
        g = gen(77)
        self.ex = Experts(E, H, I, "silu", False, 78)
        self.layer = self.ex.layer(K)
        self.router = randn(g, E, H) / H ** 0.5
        self.norm = 1 + 0.2 * randn(g, H)
        self.gu = i8.I8MatMul(i8.I8Matrix.from_float(randn(g, 2 * I, H) / H ** 0.5))
        self.down = i8.I8MatMul(i8.I8Matrix.from_float(randn(g, H, I) / I ** 0.5))
        self.I = I

    def __call__(self, x, residual):
        rows, total, y = i8.rmsnorm_i8(x, self.norm, 1e-6, residual=residual, keep_y=True)
        out, ids, w = self.layer.forward(rows, ops.router_logits(self.router, y), x.dtype)
        gu = self.gu(rows, x.dtype)
        shared = self.down(i8.swiglu_i8(gu[:, :self.I], gu[:, self.I:]), x.dtype)
        return total, out, shared, ids


def block_inputs(T, seed, H=640):
    g = gen(seed)
    return make_rows(g, T, H).to(torch.bfloat16), randn(g, T, H).to(torch.bfloat16)


def expert64(y, dy, wg, wu, wd):
    """down(silu(gate y) up y) in 64-bit floats, and how far off it may be when y is off by dy an element and h is rounded to codes:
    |silu'| <= 1.1 and |silu(v)| <= |v|, a code is off by half a step, a step is max|h| / 127."""
    g, u = y @ wg.t(), y @ wu.t()
    dg, du = dy @ wg.abs().t(), dy @ wu.abs().t()
    h = glu64(g, u, ACTS["silu"])
    dh = 1.1 * dg * (u.abs() + du) + g.abs() * du
    dh = dh + (h.abs() + dh).amax(-1, keepdim=True) / 254
    return h @ wd.t(), dh @ wd.abs().t()


@pytest.mark.parametrize("T", [1, 5, 70])
def test_block_follows_floats(T):
    """The whole block against 64-bit floats without any rounding to codes (the weights are what their codes stand for): within what
    half a step of y and of h make at most of the outputs, and 1 % of that and of the output for the roundings to bf16 on the way
    (2^-9 each) and f32."""
    b = Block()
    x, r = block_inputs(T, 5)
    total, out, shared, ids = b(x, r)
    h = (x.float() + r.float()).to(x.dtype)
    assert torch.equal(total, h)
    y = h.double() / torch.sqrt(h.double().square().mean(1, keepdim=True) + 1e-6) * b.norm.double()
    dy = (y.abs().amax(1, keepdim=True) / 254).expand_as(y)
    p = torch.softmax(y @ b.router.double().t(), 1).gather(1, ids.long())
    p = p / p.sum(1, keepdim=True)
    want, off = torch.zeros_like(y), torch.zeros_like(y)
    for t in range(T):
        for j in range(ids.shape[1]):
            v, d = expert64(y[t], dy[t], *[q[ids[t, j]].double()[:, :k] * s[ids[t, j]].double()[:, None] for q, s, k in b.ex.w])
            want[t] += p[t, j] * v
            off[t] += p[t, j] * d
    assert ((out.double() - want).abs() <= 1.01 * off + 0.01 * want.abs()).all()
    gu, down = (m.w.q.double()[:, :m.w.k] * m.w.scale.double()[:, None] for m in (b.gu, b.down))
    want, off = expert64(y, dy, gu[:b.I], gu[b.I:], down)
    assert ((shared.double() - want).abs() <= 1.01 * off + 0.01 * want.abs()).all()


@pytest.mark.parametrize("T", [1, 70])
def test_block_step_by_step(T):
    """Each step of the block on what the step before it gave."""
    b = Block()
    x, r = block_inputs(T, 6)
    rows, total, y = i8.rmsnorm_i8(x, b.norm, 1e-6, residual=r, keep_y=True)
    logits = ops.router_logits(b.router, y)
    out, ids, w = b.layer.forward(rows, logits, x.dtype)
    b.ex.check((rows.q, rows.scale), logits, 4, True, out, ids, w)
    gu = b.gu(rows, x.dtype)
    check_matmul((rows.q, rows.scale), (b.gu.w.q, b.gu.w.scale), None, x.dtype, gu)
    h = i8.swiglu_i8(gu[:, :b.I], gu[:, b.I:])
    v = gu.double()
    assert v[:, :b.I].abs().max() < 16  # of silu's error in f32 only exp's and the sums' and products' own count
    check_codes(h, glu64(v[:, :b.I], v[:, b.I:], ACTS["silu"]), GLU_REL)
    shared = b.down(h, x.dtype)
    check_matmul((h.q, h.scale), (b.down.w.q, b.down.w.scale), None, x.dtype, shared)
    got = b(x, r)
    assert all(torch.equal(p, q) for p, q in zip(got, (total, out, shared, ids)))


@pytest.mark.parametrize("T", [1, 33])
def test_block_in_two_graphs_replayed_with_new_inputs(T):
    b = Block()
    x, r = block_inputs(T, 1)
    b(x, r)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr, xi, ri = torch.cuda.CUDAGraph(), x.clone(), r.clone()
        with torch.cuda.graph(gr):
            outs = b(xi, ri)
        graphs.append((gr, xi, ri, outs))
    for n in range(4):
        for k, (gr, xi, ri, outs) in enumerate(graphs):
            nx, nr = block_inputs(T, 10 + 2 * n + k)
            xi.copy_(nx)
            ri.copy_(nr)
        for gr, *_ in graphs:
            gr.replay()
        wants = [b(xi, ri) for _, xi, ri, _ in graphs]
        torch.cuda.synchronize()
        for (_, _, _, outs), want in zip(graphs, wants):
            assert all(torch.equal(o, v) for o, v in zip(outs, want))


@pytest.mark.parametrize("T", [1, 40])
def test_block_on_streams_at_once(T):
    b = Block()
    ins = [block_inputs(T, s) for s in range(4)]
    want = [b(*v) for v in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = []
    for v, st in zip(ins, streams):
        with torch.cuda.stream(st):
            got.append(b(*v))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_no_rows():
    b = Block()
    total, out, shared, ids = b(*[v[:0] for v in block_inputs(1, 1)])
    assert total.shape == out.shape == shared.shape == (0, 640) and ids.shape == (0, 4)


def test_refusals():
    g = gen(4)
    x = randn(g, 4, 256)
    rows = i8.quantize_i8(x)
    m = i8.I8Matrix.from_float(randn(g, 8, 256))
    bad = [lambda: i8.quantize_i8(x.double()), lambda: i8.quantize_i8(x.cpu()), lambda: i8.quantize_i8(x.t()), lambda: i8.quantize_i8(x[0]),
           lambda: i8.quantize_i8(torch.empty(1, 40000, device="cuda")), lambda: i8.quantize_i8(x[:1].expand(4, 256)),
           lambda: i8.swiglu_i8(x, x[:, :128]), lambda: i8.swiglu_i8(x, x.half()),
           lambda: i8.swiglu_i8(x, x, ops.ExpertAct.clamped_swiglu(1.0, 7.0, x, None, None)),
           lambda: i8.rmsnorm_i8(x, x[0, :100].contiguous(), 1e-6), lambda: i8.rmsnorm_i8(x, x[0].contiguous(), 1e-6, residual=x[:2]),
           lambda: i8.rmsnorm_i8(x, x[0].contiguous(), -1.0), lambda: i8.rmsnorm_i8(x, x[0].contiguous(), 1e-6, residual=x.half()),
           lambda: i8.I8MatMul(m, x[0].contiguous()), lambda: i8.I8MatMul(m)(i8.quantize_i8(x[:, :100])), lambda: i8.I8MatMul(m)(rows, torch.float64),
           lambda: i8.I8Rows(rows.q, rows.scale, 100), lambda: i8.I8Rows(rows.q, rows.scale[:2], 256), lambda: i8.I8Rows(rows.q.float(), rows.scale, 256),
           lambda: i8.I8Rows(rows.q.view(-1)[128:-128].view(-1, 256), rows.scale, 256),
           lambda: rows.dequantize(torch.float64)]
    ex = Experts(4, 256, 64, "silu", False, 1)
    layer, logits = ex.layer(2), randn(g, 4, 4)
    bad += [lambda: layer.forward(rows, logits[:, :3].contiguous()), lambda: layer.forward(i8.quantize_i8(x[:, :128]), logits),
            lambda: layer.forward(rows, logits.half()), lambda: layer.forward(rows, logits, torch.float64),
            lambda: ex.layer(5).forward(rows, logits), lambda: ex.layer(0).forward(rows, logits),
            lambda: i8.I8MoeLayer(*[i8.I8ExpertBank(*ex.w[i]) for i in (0, 2, 1)], top_k=2)]
    for n, call in enumerate(bad):
        with pytest.raises(cw.CwError):
            call()
            say("not refused:", n)
    torch.cuda.synchronize()
