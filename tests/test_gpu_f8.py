"""Experts in 8-bit floats against the same formulas in 64 bits.

A code is the nearest e4m3 value, so it may differ from the oracle's only where the value lies as near to the border between two codes
as its own error. A product's sums are f32: 128 products by the matrix instruction, taken to be off by a step (2 U) for each, and a
rounding for each block of 128 and each wave that joins them."""
import itertools

import pytest
import torch

import coachwhip_amd as cw
from coachwhip_amd import f8, ops, piles, synth
from coachwhip_amd import formats as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24  # half a step of f32
E4M3 = torch.float8_e4m3fn


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def say(*a):
    print(*a, flush=True)


def step_of(t):
    """The distance between neighbouring e4m3 values about t."""
    return torch.exp2(torch.clamp(torch.frexp(t.abs()).exponent - 1, min=-6).double() - 3)


def grouped(y):
    """(rows, k) -> (rows, blocks, 128), zeros past k."""
    out = y.new_zeros((y.shape[0], f8.blocks(y.shape[1]) * 128))
    out[:, :y.shape[1]] = y
    return out.view(y.shape[0], -1, 128)


def check_codes(rows, y, rel):
    """rows against y in 64 bits, whose f32 values are off by rel of themselves at most: scales by rel and their rounding, codes by
    2 rel of their value (their value's error and that of the largest) and the rounding of the quotient before they are rounded."""
    assert rows.q.shape[1] == f8.row_bytes(rows.k) and not rows.q[:, rows.k:].view(torch.uint8).any()
    g = grouped(y)
    a = g.abs().amax(2)
    s = rows.scale.t().double()
    assert ((s - a / 448).abs() <= (rel + U) * a / 448 + 2.0 ** -150).all()
    t = g * (448 / a.clamp(min=1e-300))[..., None]
    got = rows.q.double().view(g.shape)
    near = (2 * rel + U) * t.abs()
    assert ((got - t).abs() <= step_of(t + near) / 2 + near).all()


def values(rows):
    return (rows.q.double().view(len(rows), -1, 128) * rows.scale.t().double()[..., None]).view(len(rows), -1)[:, :rows.k]


def matrix_values(q, scale, k):
    n = q.shape[0]
    return q[:, :k].double() * scale.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def make_rows(g, n, k, loud=4):
    x = randn(g, n, k)
    x[:, :: max(1, k // loud)] *= 9
    return x


def rand_codes(g, *shape, k):
    q = torch.zeros((*shape, f8.row_bytes(k)), device="cuda")
    q[..., :k] = randn(g, *shape, k) * 100
    return q.clamp_(-448, 448).to(E4M3)


def rand_rows(g, n, k):
    return f8.F8Rows(rand_codes(g, n, k=k), 0.001 + 0.01 * torch.rand((f8.blocks(k), n), generator=g, device="cuda"), k)


def rand_matrix(g, n, k):
    return f8.F8Matrix(rand_codes(g, n, k=k), 0.001 + 0.01 * torch.rand((f8.blocks(n), f8.blocks(k)), generator=g, device="cuda"), k)


def rand_bank(g, e, n, k):
    return f8.F8ExpertBank(rand_codes(g, e, n, k=k), 0.001 + 0.01 * torch.rand((e, f8.blocks(n), f8.blocks(k)), generator=g, device="cuda"), k)


def sums_off(k):
    """Of the sum of the terms' magnitudes: a product's sum in f32."""
    return (2 * 128 + f8.blocks(k) + 16) * U


# ------------------------------------------------------------------------------ rows to codes

ROW_SHAPES = [(1, 1), (3, 7), (1, 128), (2, 129), (5, 512), (17, 1000), (1, 2048), (16, 2880), (33, 2880), (3, 4097), (2, 8192), (2, 9001), (1, 32768), (1030, 66), (2053, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", ROW_SHAPES)
def test_quantize_matches_64_bits(rows, k, dtype):
    say("quantize", rows, k, dtype)
    x = make_rows(gen(k), rows, k).to(dtype)
    r = f8.quantize_f8(x)
    check_codes(r, x.double(), 0.0)
    want = values(r)
    for out in DTYPES:
        assert ((r.dequantize(out).double() - want).abs() <= half(out) * want.abs() + U * want.abs() + torch.finfo(out).tiny).all()


@pytest.mark.parametrize("top", [448.0, 7.0, 3.5, 238.0, 21.0, 1.0])
def test_ties_go_to_the_even_code(top):
    """Values on the border between two codes: 448 x / top is exact or its f32 rounding is, and the nearest even code is asked for."""
    mid = torch.tensor([(16 + 2 * i + 1) * 2.0 ** (e - 4) for e in range(-5, 8) for i in range(8)], dtype=torch.float64)
    x = (mid * top / 448)
    x = x[x.float().double() == x].float()[:126]
    assert x.numel() >= 13  # (tops without the factor 7 leave the one fraction of 17, 19, .. 31 that has it, 21, at 13 exponents)
    row = torch.zeros(1, 128)
    row[0, :x.numel()], row[0, 127] = x, top
    got = f8.quantize_f8(row.cuda()).q
    assert torch.equal(got.view(torch.uint8).cpu(), (row.double() * 448 / top).float().to(E4M3).view(torch.uint8))


def test_quantize_of_strided_and_unaligned_rows():
    for dtype in DTYPES:
        base = make_rows(gen(1), 40, 531).to(dtype)
        for view in (base[:, :300], base[:, 1:301], base[::2, 5:77], base[3:4, 7:]):
            r = f8.quantize_f8(view)
            want = f8.quantize_f8(view.contiguous())
            assert torch.equal(r.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(r.scale, want.scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_groups_without_a_scale(dtype):
    """Zeros, infinities, NaN and the type's extremes, a group at a time: the groups beside them keep their codes."""
    x = randn(gen(2), 6, 400).to(dtype)
    clean = f8.quantize_f8(x)
    x[0, :128] = 0
    x[1, 130] = float("inf")
    x[2, 399] = float("nan")
    x[3, 5] = -float("inf")
    x[4, 128:256] = torch.finfo(dtype).max
    x[5, 256:384] = torch.finfo(dtype).smallest_normal
    r = f8.quantize_f8(x)
    hit = {(0, 0), (1, 1), (2, 3), (3, 0), (4, 1), (5, 2)}
    for row, b in itertools.product(range(6), range(4)):
        code = r.q[row, 128 * b:128 * (b + 1)].view(torch.uint8)
        if (row, b) not in hit:
            assert torch.equal(code, clean.q[row, 128 * b:128 * (b + 1)].view(torch.uint8)) and r.scale[b, row] == clean.scale[b, row]
    assert r.scale[0, 0] == 0 and not r.q[0, :128].view(torch.uint8).any()
    for row, b in ((1, 1), (2, 3), (3, 0)):
        assert r.scale[b, row].isnan() and not r.q[row, 128 * b:128 * (b + 1)].view(torch.uint8).any()
    assert (r.q[4, 128:256].float() == 448).all() and (r.q[5, 256:384].float() == 448).all()
    assert r.dequantize(dtype)[1, 128:256].isnan().all() and not r.dequantize(dtype)[1, :128].isnan().any()


def glu64(g, u, act):
    if act.kind == 0:
        return g * torch.sigmoid(g) * u
    g, u = g.clamp(max=act.limit), u.clamp(-act.limit, act.limit)
    return (u + 1) * g * torch.sigmoid(act.alpha * g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [ops.ExpertAct.silu(), ops.ExpertAct.clamped_swiglu(1.702, 7.0, None, None, None)])
@pytest.mark.parametrize("rows,k", [(1, 512), (7, 129), (33, 2880), (300, 77)])
def test_swiglu_matches_64_bits(rows, k, act, dtype):
    say("swiglu", rows, k, dtype, act.kind)
    gu = (2 * randn(gen(k), rows, 2 * k + 3)).to(dtype)
    g, u = gu[:, :k], gu[:, k + 3:]
    r = f8.swiglu_f8(g, u, act)
    # the activation: 9 half steps of f32; the clamped form's sum u + 1, of a u that f32 holds, is rounded once
    check_codes(r, glu64(g.double(), u.double(), act), 12 * U)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 257), (300, 2880), (2048, 130)])
def test_matrices_match_64_bits(n, k, dtype):
    w = (0.05 * make_rows(gen(n), n, k)).to(dtype)
    m = f8.F8Matrix.from_float(w)
    assert not m.q[:, k:].view(torch.uint8).any() and m.shape == (n, k)
    for nb, kb in itertools.product(range(f8.blocks(n)), range(f8.blocks(k))):
        y = w[128 * nb:128 * (nb + 1), 128 * kb:128 * (kb + 1)].double()
        a = y.abs().max()
        assert abs(m.scale[nb, kb].double() - a / 448) <= U * a / 448
        t = y * 448 / a
        got = m.q[128 * nb:128 * nb + y.shape[0], 128 * kb:128 * kb + y.shape[1]].double()
        assert ((got - t).abs() <= step_of(t * (1 + U)) / 2 + U * t.abs()).all()


def test_matrices_of_gguf_weights():
    g = torch.Generator().manual_seed(1)
    raw = torch.randint(0, 256, (64 * 256 // 32 * 34,), generator=g, dtype=torch.uint8).view(-1, 34)
    raw[:, 0], raw[:, 1] = 0, 0x20  # an f16 scale of 2^-7
    q = ops.QTensor(raw.reshape(-1).cuda(), F.Q8_0, (64, 256))
    got, want = f8.F8Matrix.from_qtensor(q), f8.F8Matrix.from_float(q.dequantize())
    assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.scale, want.scale)
    bank = ops.ExpertBank(q.data, F.Q8_0, 32, 256, 2, 32 * 256 // 32 * 34)
    b = f8.F8ExpertBank.from_bank(bank)
    whole = f8.F8ExpertBank.from_float(q.dequantize().view(2, 32, 256))
    assert torch.equal(b.q.view(torch.uint8), whole.q.view(torch.uint8)) and torch.equal(b.scale, whole.scale)


# ------------------------------------------------------------------------------ products

MATMUL_SHAPES = [(1, 1, 1), (1, 2048, 2048), (3, 17, 130), (16, 100, 4096), (17, 333, 1000), (32, 512, 2880), (33, 640, 512), (64, 1000, 300), (65, 200, 129),
                 (77, 4001, 2880), (100, 64, 128), (129, 129, 640), (200, 2000, 2880), (513, 1027, 257), (300, 4096, 4096), (2049, 4097, 1000), (1500, 700, 32768), (4100, 2900, 385)]


def check_product(y, x, w, bias, dtype, k):
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    # results in f16 and bf16 come from the instruction on 8-bit codes, which keeps of the products of 8 neighbouring codes 18 bits below the
    # largest: each of the 8 is off by 2^-18 of the largest at most, which is at most the sum of their magnitudes: 8 * 2^-18 of it
    off = (sums_off(k) + (0.0 if dtype == torch.float32 else 2.0 ** -15)) * size
    if bias is not None:
        want, off = want + bias.double(), off + U * (want.abs() + bias.double().abs())
    assert y.dtype == dtype and y.shape == want.shape
    assert ((y.double() - want).abs() <= off + half(dtype) * (want.abs() + off) + torch.finfo(dtype).tiny).all()
    if y.numel() > 1000:
        # together: of the terms' random errors a root remains
        assert (y.double() - want).norm() <= (1e-6 if dtype == torch.float32 else half(dtype)) * want.norm()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", MATMUL_SHAPES)
def test_matmul_matches_64_bits(m, n, k, dtype, bias):
    say("matmul", m, n, k, dtype, bias)
    g = gen(m + n + k)
    x, w = rand_rows(g, m, k), rand_matrix(g, n, k)
    b = randn(g, n) if bias else None
    check_product(f8.F8MatMul(w, b)(x, dtype), values(x), matrix_values(w.q, w.scale, k), b, dtype, k)


@pytest.mark.parametrize("m", [1, 20, 40, 100, 300, 2100])
def test_scales_of_any_size(m):
    """Scales whose product leaves f32's range while the result does not, zeros, infinities and NaN, each in its own rows and columns; the rows
    and columns beside them keep their bits."""
    n, k = 300, 384
    g = gen(m)
    x, w = rand_rows(g, m, k), rand_matrix(g, n, k)
    y = f8.F8MatMul(w)(x)
    sx, sw = x.scale.clone(), w.scale.clone()
    sx[:, 0] *= 2.0 ** 100
    sw[1] *= 2.0 ** -100
    got = f8.F8MatMul(f8.F8Matrix(w.q, sw, k))(f8.F8Rows(x.q, sx, k))
    check_product(got[:, 128:256], values(f8.F8Rows(x.q, sx, k)), matrix_values(w.q, sw, k)[128:256], None, torch.float32, k)
    assert torch.equal(got[1:, :128], y[1:, :128]) and torch.equal(got[1:, 256:], y[1:, 256:])
    tiny = f8.F8MatMul(f8.F8Matrix(w.q, w.scale * 2.0 ** -70, k))(f8.F8Rows(x.q, x.scale * 2.0 ** -50, k))
    off = sums_off(k) * (values(x).abs() @ matrix_values(w.q, w.scale, k).abs().t()) * 2.0 ** -120
    assert ((tiny.double() - values(x) @ matrix_values(w.q, w.scale, k).t() * 2.0 ** -120).abs() <= off + 2.0 ** -148).all()
    if m < 4:
        return
    sx = x.scale.clone()
    sx[0, 0], sx[1, 1], sx[2, 2] = 0, float("inf"), float("nan")
    got = f8.F8MatMul(w)(f8.F8Rows(x.q, sx, k))
    assert torch.equal(got[3:], y[3:]) and got[2].isnan().all() and not got[1].isfinite().any()
    x0 = values(f8.F8Rows(x.q, sx, k))[:1]
    check_product(got[:1], x0, matrix_values(w.q, w.scale, k), None, torch.float32, k)


def test_codes_that_are_not_numbers():
    x, w = rand_rows(gen(1), 70, 256), rand_matrix(gen(2), 200, 256)
    y = f8.F8MatMul(w)(x)
    x.q.view(torch.uint8)[5, 7], w.q.view(torch.uint8)[9, 200] = 0x7F, 0xFF
    got = f8.F8MatMul(w)(x)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[5], bad[:, 9] = True, True
    assert got[bad].isnan().all() and torch.equal(got[~bad], y[~bad])


# ------------------------------------------------------------------------------ sorted rows


def check_experts(t, e, k_picks, n, k, dtype, bias, by_token, ids):
    g = gen(t + n + k)
    bank = rand_bank(g, e, n, k)
    b = randn(g, e, n) if bias else None
    p = piles.sort_picks(ids, e)
    x = rand_rows(g, t if by_token else t * k_picks, k)
    y = f8.F8ExpertMatMul(bank, b).forward(x, p, dtype, by_token=by_token)
    assert y.shape == (t * k_picks, n) and y.dtype == dtype
    xv, offsets = values(x), p.offsets.tolist()
    for i in range(e):
        at = slice(offsets[i], offsets[i + 1])
        if at.start == at.stop:
            continue
        rows = xv[p.order[at].long() // k_picks] if by_token else xv[at]
        check_product(y[at], rows, matrix_values(bank.q[i], bank.scale[i], k), None if b is None else b[i], dtype, k)
    assert (y[offsets[e]:] == 0).all()


@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,e,kp,n,k", [(1, 1, 1, 1, 1), (1, 8, 2, 128, 128), (1, 256, 8, 1024, 2048), (8, 64, 6, 300, 1000), (40, 4, 2, 129, 640), (129, 3, 1, 260, 257), (301, 16, 4, 513, 2880),
                                        (700, 5, 3, 100, 130), (1100, 2, 2, 385, 512), (2048, 32, 4, 640, 384)])
def test_experts_match_64_bits(t, e, kp, n, k, dtype, by_token):
    say("experts", t, e, kp, n, k, dtype, by_token)
    ids = torch.randint(-1, e, (t, kp), generator=gen(t), device="cuda", dtype=torch.int32)
    check_experts(t, e, kp, n, k, dtype, t % 2 == 1, by_token, ids)


@pytest.mark.parametrize("pick", [-1, 0, 6])
@pytest.mark.parametrize("t", [1, 16, 17, 33, 65, 128, 129, 300])
def test_all_on_one_expert(t, pick):
    say("one expert", t, pick)
    check_experts(t, 7, 1, 200, 300, torch.bfloat16, True, False, torch.full((t, 1), pick, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------------------ the layer


def check_layer(t, e, kp, h, i, dtype, act, norm=True, seed=0):
    # the 8-bit instruction's products (check_product) make gate and up of bf16 results, and down of bf16 and f16 ones
    less = [2.0 ** -15 if dtype == torch.bfloat16 else 0.0, 0.0 if dtype == torch.float32 else 2.0 ** -15]
    g = gen(seed + t + h)
    banks = [rand_bank(g, e, *s) for s in ((i, h), (i, h), (h, i))]
    for b in banks:
        b.scale.mul_(0.3 / b.k ** 0.5)
    biases = [0.05 * randn(g, e, n) for n in (i, i, h)] if act else [None] * 3
    act = ops.ExpertAct.clamped_swiglu(1.702, 7.0, *biases) if act else ops.ExpertAct.silu()
    layer = f8.F8MoeLayer(*banks, top_k=kp, norm_topk_prob=norm, act=act)
    x, logits = f8.quantize_f8(randn(g, t, h)), randn(g, t, e)
    out, ids, w = layer.forward(x, logits, dtype)
    wids, ww = ops.route(logits, kp, norm)
    assert torch.equal(ids, wids) and torch.equal(w, ww) and out.dtype == dtype and out.shape == (t, h)
    xv = values(x)
    want, off = torch.zeros(t, h, dtype=torch.float64, device="cuda"), torch.zeros(t, h, dtype=torch.float64, device="cuda")
    for x_ in range(e):
        tok, j = torch.nonzero(ids == x_, as_tuple=True)
        if not tok.numel():
            continue
        gate, up, down = (matrix_values(b.q[x_], b.scale[x_], b.k) for b in banks)
        gb, ub, db = (0.0 if b is None else b[x_].double() for b in biases)
        gv, uv = xv[tok] @ gate.t() + gb, xv[tok] @ up.t() + ub
        ge, ue = ((sums_off(h) + less[0]) * (xv[tok].abs() @ m.abs().t()) + 2 * U * v.abs() for m, v in ((gate, gv), (up, uv)))
        hv = glu64(gv, uv, act)
        # the activation's slope in g is at most 1.1 |u| (2 |u + 1| of the clamped form), in u |silu(g)| <= |g|; its own roundings
        he = ge * 2 * (uv.abs() + 1) + ue * gv.abs() + 12 * U * (gv.abs() * (uv.abs() + 1))
        G, H = grouped(hv), grouped(he)
        a, ae = G.abs().amax(2, keepdim=True), H.amax(2, keepdim=True)
        tq = (G * 448 / a.clamp(min=1e-300)).float().double()
        step = step_of(tq)
        code = torch.round(tq / step) * step
        # how far the code's value may be: a step where the value's error (its own and the largest's) reaches the border, and the scale's error
        te = 448 * (H / a + G.abs() * ae / a ** 2) + U * tq.abs()
        border = step / 2 - (tq - code).abs()
        far = torch.where(border <= te, step, 0.0)
        hq, s = (code * a / 448).view(hv.shape[0], -1)[:, :i], a / 448
        ho = (far * s + code.abs() * s * (U + ae / a)).view(hv.shape[0], -1)[:, :i]
        y = hq @ down.t() + db
        yo = ho @ down.abs().t() + (sums_off(i) + less[1]) * (hq.abs() @ down.abs().t()) + U * y.abs()
        wt = w[tok, j].double()[:, None]
        want.index_add_(0, tok, wt * y)
        off.index_add_(0, tok, wt * (yo + 2 * U * kp * y.abs()))
    assert ((out.double() - want).abs() <= off + half(dtype) * (want.abs() + off) + torch.finfo(dtype).tiny).all()
    return layer, x, logits, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("t,e,kp,h,i", [(1, 8, 2, 128, 128), (1, 256, 8, 2048, 512), (3, 40, 6, 300, 77), (8, 64, 8, 1000, 129), (16, 8, 1, 2880, 640), (33, 512, 10, 256, 256),
                                        (130, 16, 4, 513, 300), (700, 4, 2, 384, 1000)])
def test_layer_matches_64_bits(t, e, kp, h, i, act, dtype):
    say("layer", t, e, kp, h, i, act, dtype)
    check_layer(t, e, kp, h, i, dtype, act, norm=t % 2 == 0)


@pytest.mark.parametrize("t", [2, 40, 300])
def test_a_token_that_is_not_finite_stays_alone(t):
    layer, x, logits, out = check_layer(t, 16, 4, 256, 200, torch.float32, True)
    x.scale[1, 1] = float("nan")
    got, _, _ = layer.forward(x, logits)
    keep = torch.arange(t, device="cuda") != 1
    assert got[1].isnan().all() and torch.equal(got[keep], out[keep])


def test_no_tokens():
    g = gen(0)
    bank = rand_bank(g, 4, 200, 300)
    empty = f8.quantize_f8(torch.empty(0, 300, device="cuda"))
    assert empty.dequantize().shape == (0, 300) and f8.F8MatMul(rand_matrix(g, 200, 300))(empty).shape == (0, 200)
    p = piles.sort_picks(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 4)
    assert p.offsets.tolist() == [0] * 5 and f8.F8ExpertMatMul(bank)(empty, p).shape == (0, 200)
    layer = f8.F8MoeLayer(bank, rand_bank(g, 4, 200, 300), rand_bank(g, 4, 300, 200), top_k=2)
    out, ids, w = layer.forward(empty, torch.empty(0, 4, device="cuda"))
    assert out.shape == (0, 300) and ids.shape == w.shape == (0, 2)


# ------------------------------------------------------------------------------ streams, graphs, refusals


@pytest.mark.parametrize("t", [1, 8, 300])
def test_captured_and_replayed(t):
    """Rows to codes, the sort, the experts' product, the way back and the layer in one graph, replayed on other inputs between eager runs."""
    e, kp, h, i = 32, 4, 512, 384
    g = gen(t)
    x, logits = randn(g, t, h).bfloat16(), randn(g, t, e)
    bank, layer = rand_bank(g, e, h, h), f8.F8MoeLayer(rand_bank(g, e, i, h), rand_bank(g, e, i, h), rand_bank(g, e, h, i), top_k=kp)

    def run():
        rows = f8.quantize_f8(x)
        ids, w = ops.route(logits, kp, True)
        p = piles.sort_picks(ids, e)
        y = f8.F8ExpertMatMul(bank)(rows, p, torch.bfloat16, by_token=True)
        out = piles.from_piles(y, w, p)
        return y, out, layer.forward(f8.quantize_f8(out), logits, torch.bfloat16)[0], f8.F8MatMul(rand)(f8.quantize_f8(out))

    rand = rand_matrix(g, 100, h)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in (1, 2, 3):
        x.copy_(randn(gen(seed), t, h))
        logits.copy_(randn(gen(seed + 9), t, e))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, run()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_on_a_stream_of_its_own():
    g = gen(4)
    x, w = rand_rows(g, 300, 512), rand_matrix(g, 700, 512)
    want = f8.F8MatMul(w)(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = f8.F8MatMul(w)(x)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(got, want)


def test_refusals():
    g = gen(0)
    x, w, bank = rand_rows(g, 6, 256), rand_matrix(g, 100, 256), rand_bank(g, 3, 100, 256)
    p = piles.sort_picks(torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 3)
    f = torch.randn(6, 256, device="cuda")
    bad = [lambda: f8.quantize_f8(f.double()), lambda: f8.quantize_f8(f.t()), lambda: f8.quantize_f8(f[0]), lambda: f8.quantize_f8(f[:, :0]),
           lambda: f8.swiglu_f8(f, f[:, :100]), lambda: f8.swiglu_f8(f, f.half()), lambda: f8.swiglu_f8(f, f, ops.ExpertAct(gate_b=f)),
           lambda: f8.F8Rows(x.q, x.scale.t(), 256), lambda: f8.F8Rows(x.q, x.scale, 100),
           lambda: f8.F8Rows(x.q.view(torch.uint8), x.scale, 256), lambda: f8.F8Rows(x.q, x.scale.t().contiguous(), 256),
           lambda: f8.F8Rows(x.q.view(torch.uint8).view(torch.float8_e5m2), x.scale, 256), lambda: f8.F8Matrix(w.q, x.scale, 256), lambda: f8.F8Matrix(w.q, w.scale.double(), 256),
           lambda: f8.F8ExpertBank(bank.q, w.scale, 256), lambda: f8.F8MatMul(w, torch.zeros(99, device="cuda")), lambda: f8.F8MatMul(w)(rand_rows(g, 2, 128)),
           lambda: f8.F8MatMul(w)(x, torch.float64), lambda: x.dequantize(torch.int8), lambda: f8.F8ExpertMatMul(bank, torch.zeros(3, 99, device="cuda")),
           lambda: f8.F8ExpertMatMul(bank)(x, p, by_token=True), lambda: f8.F8ExpertMatMul(bank)(rand_rows(g, 3, 256), p),
           lambda: f8.F8ExpertMatMul(rand_bank(g, 4, 100, 256))(x, p), lambda: f8.F8ExpertMatMul(bank)(x, p, torch.int8),
           lambda: f8.F8MoeLayer(bank, bank, bank, top_k=1), lambda: f8.F8MoeLayer(bank, bank, rand_bank(g, 3, 256, 100), top_k=4).forward(x, torch.zeros(6, 3, device="cuda")),
           lambda: f8.F8MoeLayer(bank, bank, rand_bank(g, 3, 256, 100), top_k=2).forward(x, torch.zeros(5, 3, device="cuda"))]
    for call in bad:
        with pytest.raises(cw.CwError):
            call()
    assert f8.F8MatMul(w)(x).shape == (6, 100)


@pytest.mark.parametrize("t", [2, 40, 700])
def test_layer_with_strange_scales(t):
    """Scales of gate, up and down whose product with the rows' leaves f32 while the results do not."""
    e, kp, h, i = 8, 2, 300, 260
    g = gen(t)
    banks = [rand_bank(g, e, *s) for s in ((i, h), (i, h), (h, i))]
    for b in banks:
        b.scale.mul_(0.3 / b.k ** 0.5)
    x, logits = f8.quantize_f8(randn(g, t, h)), randn(g, t, e)
    want, _, _ = f8.F8MoeLayer(*banks, top_k=kp).forward(x, logits)
    big = 2.0 ** 70
    for b in banks[:2]:
        b.scale.div_(big)
    got, _, _ = f8.F8MoeLayer(*banks, top_k=kp).forward(f8.F8Rows(x.q, x.scale * big, h), logits)
    # the same numbers, added in another order: what a hidden code's step makes of it, 2^-4 of a value for one of many
    assert (got - want).norm() <= 2e-3 * want.norm()
