"""The 8-bit integer path of a mixture-of-experts block, as cases that can be timed and compared.

Four operators, each with its plain form (elementary torch operations) and, where `own` is true, the package's:
- norm: RMS norm with the residual's addition, its rows out as 8-bit codes with a scale each;
- swiglu: silu(g) u (or the clamped form of gpt-oss's experts) of two halves of a projection, as 8-bit rows;
- matmul: 8-bit rows times an 8-bit matrix, a scale for each row and each output channel;
- moe: a layer of 8-bit experts on 8-bit rows: routing, gate and up, the activation, down, the weighted sum.

8-bit rows are held as the package holds them: k codes, zeros up to the next multiple of 128 bytes, and a scale a row.
Codes come back as the values that they stand for, in the type of the activations.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}

# ------------------------------------------------------------------------------ the cases


def _norm(name, dtype, rows, k, residual=True, keep=False):
    return {"name": name, "kind": "norm", "dtype": dtype, "rows": rows, "k": k, "residual": residual, "keep": keep}


def _swiglu(name, dtype, rows, width, act="silu"):
    return {"name": name, "kind": "swiglu", "dtype": dtype, "rows": rows, "width": width, "act": act}


def _matmul(name, dtype, m, n, k, bias=False):
    return {"name": name, "kind": "matmul", "dtype": dtype, "m": m, "n": n, "k": k, "bias": bias}


def _moe(name, dtype, tokens, experts, top_k, hidden, inter, act="silu"):
    return {"name": name, "kind": "moe", "dtype": dtype, "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden,
            "inter": inter, "act": act}


def listed():
    return [
        # one token before a layer's experts: the router reads the norm's f32 rows, the experts its codes
        _norm("norm_1token", "f32", 1, 2048, keep=True),
        # a short prompt of odd length in a model of width 2,880
        _norm("norm_301tokens", "bf16", 301, 2880, keep=True),
        # a batch of prompts
        _norm("norm_8192tokens", "bf16", 8192, 4096),
        # the shared expert's activation for 64 sequences decoded together
        _swiglu("swiglu_64rows", "f16", 64, 512),
        # the clamped activation over the picks of 2,048 tokens
        _swiglu("swiglu_8192rows", "bf16", 8192, 2880, "clamped"),
        # the smallest product: one token through a small projection
        _matmul("matmul_1row", "bf16", 1, 2048, 2048),
        # 16 sequences decoded together through an attention-sized projection
        _matmul("matmul_16rows", "bf16", 16, 4096, 4096),
        # a short prompt through a matrix of odd sizes, with a bias
        _matmul("matmul_77rows", "f32", 77, 4001, 2880, True),
        # a batch of prompts: the largest product
        _matmul("matmul_8192rows", "bf16", 8192, 4096, 4096),
        # one token through 256 small experts, top-8
        _moe("moe_1token", "bf16", 1, 256, 8, 2048, 512),
        # 8 sequences decoded together
        _moe("moe_8tokens", "bf16", 8, 256, 8, 2048, 512),
        # a prompt of 2,048 tokens through 128 wide experts with biases, top-4
        _moe("moe_2048tokens", "bf16", 2048, 128, 4, 2880, 2880, "clamped"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "swiglu", "matmul", "matmul", "moe", "moe"])
    if kind == "norm":
        k = _log_int(rng, 64, 8192)
        c = _norm("", rng.choice(list(_TYPES)), _log_int(rng, 1, min(8192, 8192 * 2048 // k)), k, rng.random() < 0.75, rng.random() < 0.5)
    elif kind == "swiglu":
        width = _log_int(rng, 64, 8192)
        c = _swiglu("", rng.choice(["f16", "bf16"]), _log_int(rng, 1, min(8192, 8192 * 2880 // width)), width, rng.choice(["silu", "clamped"]))
    elif kind == "matmul":
        n, k = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
        c = _matmul("", rng.choice(list(_TYPES)), _log_int(rng, 1, min(8192, 8192 * 4096 * 2048 // (n * k))), n, k, rng.random() < 0.5)
    else:
        top_k, hidden, inter = rng.randint(1, 10), _log_int(rng, 128, 4096), _log_int(rng, 64, 2880)
        experts = _log_int(rng, max(8, top_k), min(512, max(10, int(1e9 / (hidden * inter)))))
        tokens = _log_int(rng, 1, min(2048, int(8192 * 2880 * 2880 / (top_k * hidden * inter))))
        c = _moe("", rng.choice(["f16", "bf16"]), tokens, experts, top_k, hidden, inter, rng.choice(["silu", "clamped"]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------ inputs (of the seed alone)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _row_bytes(k):
    return (k + 127) // 128 * 128


def _activations(gen, rows, k):
    """Activations as a model's: a few channels an order of magnitude above the others."""
    loud = 1 + 9 * (torch.rand(k, generator=gen, device="cuda") < 0.004)
    return _randn(gen, rows, k) * loud


def _codes(gen, lead, n, k):
    """n rows of k codes of normal weights whose largest is about 127, in rows of whole 128 bytes, and a scale a row."""
    q = torch.zeros((*lead, n, _row_bytes(k)), dtype=torch.int8, device="cuda")
    q[..., :k] = (_randn(gen, *lead, n, k) * 31).round_().clamp_(-127, 127)
    return q, (0.5 + torch.rand((*lead, n), generator=gen, device="cuda")) / (31 * math.sqrt(k))


def _rows(x):
    """Activations as 8-bit rows: what a program holds after the layer before."""
    rows, k = x.shape
    scale = x.abs().amax(1) / 127
    q = torch.zeros((rows, _row_bytes(k)), dtype=torch.int8, device="cuda")
    q[:, :k] = (x / scale[:, None]).round()
    return q, scale


def _inputs(c, seed):
    gen, d = _gen(seed), {}
    dtype = _TYPES[c["dtype"]]
    if c["kind"] == "norm":
        d["x"] = _activations(gen, c["rows"], c["k"]).to(dtype)
        d["residual"] = (2 * _activations(gen, c["rows"], c["k"])).to(dtype) if c["residual"] else None
        d["weight"] = 1 + 0.2 * _randn(gen, c["k"])
    elif c["kind"] == "swiglu":
        # one projection's rows: the gate's half, then the up's
        d["gu"] = (1.5 * _randn(gen, c["rows"], 2 * c["width"])).to(dtype)
    elif c["kind"] == "matmul":
        d["x"] = _rows(_activations(gen, c["m"], c["k"]))
        d["w"] = _codes(gen, (), c["n"], c["k"])
        d["bias"] = 0.1 * _randn(gen, c["n"]) if c["bias"] else None
    else:
        t, e, h, i = c["tokens"], c["experts"], c["hidden"], c["inter"]
        d["x"] = _rows(_activations(gen, t, h))
        d["logits"] = _randn(gen, t, e)
        d["w"] = [_codes(gen, (e,), n, k) for n, k in ((i, h), (i, h), (h, i))]
        d["bias"] = [0.02 * _randn(gen, e, n) for n in (i, i, h)] if c["act"] == "clamped" else None
    return d


_EPS, _ALPHA, _LIMIT = 1e-6, 1.702, 7.0

# ------------------------------------------------------------------------------ the plain forms


def _quantized(y, dtype):
    """The values that y's 8-bit rows stand for, and their scales."""
    a = y.abs().amax(1, keepdim=True)
    q = torch.round(y * (127 / a))
    scale = (a / 127).float()
    return (q.float() * scale).to(dtype), scale[:, 0]


def _act(g, u, act):
    if act == "silu":
        return g / (1 + torch.exp(-g)) * u
    g, u = g.clamp(max=_LIMIT), u.clamp(-_LIMIT, _LIMIT)
    return (u + 1) * (g / (1 + torch.exp(-_ALPHA * g)))


def _plain_norm(c, d):
    # a code is a choice between two neighbours: in 64 bits, so that it does not hang on the order of a sum
    h = d["x"] if d["residual"] is None else (d["x"].float() + d["residual"].float()).to(d["x"].dtype)
    y = h.double()
    y = y * torch.rsqrt(y.square().mean(1, keepdim=True) + _EPS) * d["weight"].double()
    values, scale = _quantized(y, h.dtype)
    out = {"values": values, "scale": scale}
    if d["residual"] is not None:
        out["sum"] = h
    if c["keep"]:
        out["y"] = y.float()
    return out


def _plain_swiglu(c, d):
    g, u = d["gu"].float().split(c["width"], 1)
    values, scale = _quantized(_act(g, u, c["act"]), d["gu"].dtype)
    return {"values": values, "scale": scale}


def _plain_matmul(c, d):
    (x, sx), (w, sw) = d["x"], d["w"]
    y = x.float() @ w.float().t() * sx[:, None] * sw
    return (y if d["bias"] is None else y + d["bias"]).to(_TYPES[c["dtype"]])


def _plain_moe(c, d):
    k, i = c["top_k"], c["inter"]
    ids = torch.sort(d["logits"], dim=1, descending=True, stable=True)[1][:, :k]
    p = torch.softmax(d["logits"], 1).gather(1, ids)
    w = p / p.sum(1, keepdim=True)
    # the picks of each expert that has any, padded to the most that one has
    used, pile = torch.unique(ids.reshape(-1), return_inverse=True)
    order = torch.argsort(pile, stable=True)
    count = torch.bincount(pile, minlength=used.numel())
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device="cuda") - (count.cumsum(0) - count)[pile[order]]
    x = d["x"][0].float() * d["x"][1][:, None]
    xp = x.new_zeros(used.numel(), int(count.max()), x.shape[1])
    xp[pile, place] = x.repeat_interleave(k, 0)

    def product(a, m):
        q, s = d["w"][m]
        y = torch.bmm(a, q[used].float().transpose(1, 2).contiguous()) * s[used][:, None]
        return y if d["bias"] is None else y + d["bias"][m][used][:, None]

    h = _act(product(xp, 0), product(xp, 1), c["act"])
    hp = h.new_zeros(*h.shape[:2], _row_bytes(i))
    hp[..., :i] = _quantized(h.reshape(-1, i), torch.float32)[0].reshape(h.shape).nan_to_num(0.0)  # rows of no pick: none
    y = product(hp, 2)[pile, place].reshape(-1, k, c["hidden"])
    return {"out": (y * w[..., None]).sum(1).to(_TYPES[c["dtype"]]), "ids": ids.int(), "w": w}


_PLAIN = {"norm": _plain_norm, "swiglu": _plain_swiglu, "matmul": _plain_matmul, "moe": _plain_moe}

# ------------------------------------------------------------------------------ the package's


def _own_norm(c, d):
    from coachwhip_amd import i8
    rows, total, y = i8.rmsnorm_i8(d["x"], d["weight"], _EPS, residual=d["residual"], keep_y=c["keep"])
    out = {"values": rows.dequantize(d["x"].dtype), "scale": rows.scale}
    if total is not None:
        out["sum"] = total
    if y is not None:
        out["y"] = y
    return out


def _own_swiglu(c, d):
    from coachwhip_amd import i8, ops
    act = ops.ExpertAct.silu() if c["act"] == "silu" else ops.ExpertAct.clamped_swiglu(_ALPHA, _LIMIT, None, None, None)
    rows = i8.swiglu_i8(d["gu"][:, :c["width"]], d["gu"][:, c["width"]:], act)
    return {"values": rows.dequantize(d["gu"].dtype), "scale": rows.scale}


def _own_matmul(c, d):
    from coachwhip_amd import i8
    x, w = i8.I8Rows(*d["x"], c["k"]), i8.I8Matrix(*d["w"], c["k"])
    return i8.I8MatMul(w, d["bias"]).forward(x, _TYPES[c["dtype"]])


def _own_moe(c, d):
    from coachwhip_amd import i8, ops
    h, i = c["hidden"], c["inter"]
    act = ops.ExpertAct.silu() if c["act"] == "silu" else ops.ExpertAct.clamped_swiglu(_ALPHA, _LIMIT, *d["bias"])
    if "layer" not in d:  # built once, as when a model is loaded
        d["layer"] = i8.I8MoeLayer(*[i8.I8ExpertBank(q, s, k) for (q, s), k in zip(d["w"], (h, h, i))], top_k=c["top_k"], act=act)
    out, ids, w = d["layer"].forward(i8.I8Rows(*d["x"], h), d["logits"], _TYPES[c["dtype"]])
    return {"out": out, "ids": ids, "w": w}


_OWN = {"norm": _own_norm, "swiglu": _own_swiglu, "matmul": _own_matmul, "moe": _own_moe}

# ------------------------------------------------------------------------------ a pass


def prepare(case, seed):
    return case, _inputs(case, seed)


def run(state):
    case, d = state
    if own:
        return _OWN[case["kind"]](case, d)
    return _PLAIN[case["kind"]](case, d)


def work(case):
    c, b = case, _BYTES[case["dtype"]]
    if c["kind"] == "norm":
        n = c["rows"] * c["k"]
        return {"bytes": n * (b * (2 + 2 * c["residual"]) + 4 * c["keep"]) + 4 * (c["k"] + c["rows"]), "flops": 10 * n}
    if c["kind"] == "swiglu":
        n = c["rows"] * c["width"]
        return {"bytes": 3 * b * n + 4 * c["rows"], "flops": 12 * n}
    if c["kind"] == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": (m + n) * (k + 4) + 4 * n * c["bias"] + b * m * n, "flops": 2 * m * n * k}
    t, e, k, h, i = c["tokens"], c["experts"], c["top_k"], c["hidden"], c["inter"]
    picked = e * (1 - (1 - k / e) ** t)  # experts that some token picks, on average
    expert = 3 * h * i + 4 * (2 * i + h) * (1 + (c["act"] == "clamped"))
    return {"bytes": picked * expert + t * (h + 4 + 4 * e + 8 * k + b * h), "flops": 6 * t * k * h * i}


# ------------------------------------------------------------------------------ the same in 64 bits


def _exact_rows(y):
    """(values, scales) of rows quantized in 64 bits."""
    top = y.abs().max(dim=1, keepdim=True).values
    step = top / 127.0
    return torch.where(top > 0, torch.round(y / step), 0.0) * step, step[:, 0]


def _exact_hidden(g, u, act):
    if act == "silu":
        return u * g * torch.sigmoid(g)
    g, u = torch.clamp(g, max=_LIMIT), torch.clamp(u, min=-_LIMIT, max=_LIMIT)
    return (1.0 + u) * g * torch.sigmoid(g * _ALPHA)


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "norm":
        h = d["x"].double()
        if c["residual"]:
            h = (h + d["residual"].double()).to(d["x"].dtype).double()  # the sum is stored in the activations' type
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / c["k"] + _EPS) * d["weight"].double()
        values, scale = _exact_rows(y)
        out = {"values": values, "scale": scale}
        if c["residual"]:
            out["sum"] = h
        if c["keep"]:
            out["y"] = y
        return out
    if c["kind"] == "swiglu":
        gu = d["gu"].double()
        values, scale = _exact_rows(_exact_hidden(gu[:, :c["width"]], gu[:, c["width"]:], c["act"]))
        return {"values": values, "scale": scale}

    def matrix(pair, e=None):
        q, s = pair if e is None else (pair[0][e], pair[1][e])
        return q.double() * s.double()[:, None]

    x = matrix(d["x"])
    if c["kind"] == "matmul":
        y = x @ matrix(d["w"]).t()
        return y if d["bias"] is None else y + d["bias"].double()
    i = c["inter"]
    best, ids = torch.sort(d["logits"].double(), dim=1, descending=True, stable=True)
    ids, w = ids[:, :c["top_k"]], torch.softmax(best[:, :c["top_k"]], 1)  # over the picks alone: the others' terms cancel
    out = torch.zeros(c["tokens"], c["hidden"], dtype=torch.float64, device="cuda")
    for e in torch.unique(ids).tolist():
        t, j = torch.nonzero(ids == e, as_tuple=True)
        b = [0.0] * 3 if d["bias"] is None else [v[e].double() for v in d["bias"]]
        g, u = (x[t] @ matrix(d["w"][m], e).t() + b[m] for m in (0, 1))
        h = _exact_rows(_exact_hidden(g, u, c["act"]))[0]
        out.index_add_(0, t, w[t, j][:, None] * (h @ matrix(d["w"][2], e)[:, :i].t() + b[2]))
    return {"out": out, "ids": None, "w": w}
