"""Experts in 8-bit floats with a scale for each block of 128, and the tokens' way to them and back, as cases that can be timed and
compared.

Five operators, each with its plain form (elementary torch operations) and, where `own` is true, the package's:
- rows: rows of floats, or of a SwiGLU, as e4m3 codes with a scale for each 128 columns;
- matmul: such rows times an e4m3 matrix with a scale for each block of 128 x 128;
- piles: tokens sorted by expert and back with their weights; backward, the gradients of both;
- experts: the product of sorted rows, each with its expert's matrix;
- layer: routing, sort, gate and up, the activation to codes, down, the weighted sum.

Codes are held as the package holds them: rows of k e4m3 codes, zeros up to the next multiple of 128 bytes; scales of rows as
(blocks of columns, rows), of matrices as (blocks of rows, blocks of columns). Codes come back as the values that they stand for, in
the type of the activations.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_B = 128  # columns of a scale
_TOP = 448.0  # the largest e4m3 value

# ------------------------------------------------------------------------------ the cases


def _rows(name, dtype, rows, k, act):
    return {"name": name, "kind": "rows", "dtype": dtype, "rows": rows, "k": k, "act": act}


def _matmul(name, dtype, m, n, k, bias=False):
    return {"name": name, "kind": "matmul", "dtype": dtype, "m": m, "n": n, "k": k, "bias": bias}


def _piles(name, dtype, tokens, experts, top_k, hidden, backward=False, absent=0.0):
    return {"name": name, "kind": "piles", "dtype": dtype, "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden,
            "backward": backward, "absent": absent}


def _experts(name, dtype, tokens, experts, top_k, n, k, by_token, bias=False):
    return {"name": name, "kind": "experts", "dtype": dtype, "tokens": tokens, "experts": experts, "top_k": top_k, "n": n, "k": k,
            "by_token": by_token, "bias": bias}


def _layer(name, dtype, tokens, experts, top_k, hidden, inter, act="silu"):
    return {"name": name, "kind": "layer", "dtype": dtype, "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden,
            "inter": inter, "act": act}


def listed():
    return [
        # one token before a projection: a launch's latency
        _rows("rows_1token", "bf16", 1, 2048, "none"),
        # the clamped activation over the picks of 2,048 tokens
        _rows("rows_8192swiglu", "bf16", 8192, 2880, "clamped"),
        # one token through a small projection
        _matmul("matmul_1row", "bf16", 1, 2048, 2048),
        # a short prompt through a matrix of odd sizes, with a bias
        _matmul("matmul_77rows", "f32", 77, 4001, 2880, True),
        # a batch of prompts: the largest product
        _matmul("matmul_8192rows", "bf16", 8192, 4096, 4096),
        # 8 sequences decoded together: a sort of 64 picks, their rows there and back
        _piles("piles_8tokens", "bf16", 8, 256, 8, 2048),
        # a batch of prompts over the experts that one of two devices holds
        _piles("piles_8192tokens", "bf16", 8192, 256, 8, 2048, absent=0.5),
        # a training step's gradients, an odd number of tokens
        _piles("piles_4095grad", "bf16", 4095, 128, 4, 2880, backward=True),
        # gate and up of 8 sequences decoded together: few picks an expert
        _experts("experts_8tokens", "bf16", 8, 256, 8, 1024, 2048, True),
        # down of a prompt of 2,048 tokens over wide experts, with biases
        _experts("experts_2048tokens", "bf16", 2048, 128, 4, 2880, 2880, False, True),
        # one token through 256 small experts, top-8
        _layer("layer_1token", "bf16", 1, 256, 8, 2048, 512),
        # a prompt of 2,048 tokens through 128 wide experts with biases, top-4
        _layer("layer_2048tokens", "bf16", 2048, 128, 4, 2880, 2880, "clamped"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rows", "matmul", "matmul", "piles", "piles", "experts", "layer"])
    dtype = rng.choice(list(_TYPES))
    if kind == "rows":
        k = _log_int(rng, 64, 8192)
        c = _rows("", dtype, _log_int(rng, 1, min(8192, 8192 * 2048 // k)), k, rng.choice(["none", "silu", "clamped"]))
    elif kind == "matmul":
        n, k = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
        c = _matmul("", dtype, _log_int(rng, 1, min(8192, 8192 * 4096 * 2048 // (n * k))), n, k, rng.random() < 0.5)
    else:
        top_k, hidden = rng.randint(1, 10), _log_int(rng, 128, 4096)
        absent = rng.choice([0.0, 0.0, 0.5, 0.75])
        if kind == "piles":
            c = _piles("", dtype, _log_int(rng, 1, min(8192, 8192 * 8 * 2048 // (2 * top_k * hidden))), _log_int(rng, max(8, top_k), 512), top_k,
                       hidden, rng.random() < 0.5, absent)
        elif kind == "experts":
            n = _log_int(rng, 64, 4096)
            experts = _log_int(rng, max(8, top_k), min(512, max(10, int(1e9 / (hidden * n)))))
            c = _experts("", dtype, _log_int(rng, 1, min(2048, int(8192 * 2880 * 2880 / (top_k * hidden * n)))), experts, top_k, n, hidden,
                         rng.random() < 0.5, rng.random() < 0.5)
        else:
            inter = _log_int(rng, 64, 2880)
            experts = _log_int(rng, max(8, top_k), min(512, max(10, int(1e9 / (hidden * inter)))))
            c = _layer("", rng.choice(["f16", "bf16"]), _log_int(rng, 1, min(2048, int(8192 * 2880 * 2880 / (top_k * hidden * inter)))), experts,
                       top_k, hidden, inter, rng.choice(["silu", "clamped"]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------ inputs (of the seed alone)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _activations(gen, rows, k):
    """Activations as a model's: a few channels an order of magnitude above the others."""
    loud = 1 + 9 * (torch.rand(k, generator=gen, device="cuda") < 0.004)
    return _randn(gen, rows, k) * loud


def _blocks(k):
    return (k + _B - 1) // _B


def _padded(q):
    """Codes in rows of whole 128 bytes."""
    out = torch.zeros((*q.shape[:-1], _blocks(q.shape[-1]) * _B), dtype=torch.uint8, device=q.device)
    out[..., :q.shape[-1]] = q.view(torch.uint8)
    return out.view(torch.float8_e4m3fn)


def _code_rows(x):
    """Activations as 8-bit rows: what a program holds after the layer before."""
    rows, k = x.shape
    y = torch.zeros((rows, _blocks(k) * _B), device="cuda")
    y[:, :k] = x
    g = y.view(rows, -1, _B)
    a = g.abs().amax(2).clamp(min=1e-20)
    q = (g * (_TOP / a)[..., None]).to(torch.float8_e4m3fn).view(rows, -1)
    return q, (a / _TOP).t().contiguous()


def _codes(gen, lead, n, k):
    """Normal weights whose largest are near 448, and a scale for each 128 x 128 of them."""
    q = (_randn(gen, *lead, n, k) * 100).clamp_(-_TOP, _TOP).to(torch.float8_e4m3fn)
    s = (0.5 + torch.rand((*lead, _blocks(n), _blocks(k)), generator=gen, device="cuda")) / (100 * math.sqrt(k))
    return _padded(q), s


def _picks(gen, tokens, experts, top_k, absent):
    """top_k different experts a token; with `absent`, those of the last experts are held by another device: -1."""
    ids = torch.rand(tokens, experts, generator=gen, device="cuda").argsort(1)[:, :top_k].int()
    held = experts - int(experts * absent)
    return torch.where(ids < held, ids, -1), held


def _inputs(c, seed):
    gen, d = _gen(seed), {}
    dtype = _TYPES[c["dtype"]]
    if c["kind"] == "rows":
        # with an activation one projection's rows: the gate's half, then the up's
        d["x"] = (_activations(gen, c["rows"], c["k"]) if c["act"] == "none" else 1.5 * _randn(gen, c["rows"], 2 * c["k"])).to(dtype)
    elif c["kind"] == "matmul":
        d["x"] = _code_rows(_activations(gen, c["m"], c["k"]))
        d["w"] = _codes(gen, (), c["n"], c["k"])
        d["bias"] = 0.1 * _randn(gen, c["n"]) if c["bias"] else None
    elif c["kind"] == "piles":
        t, k, h = c["tokens"], c["top_k"], c["hidden"]
        d["ids"], d["held"] = _picks(gen, t, c["experts"], k, c["absent"])
        d["w"] = torch.softmax(_randn(gen, t, k), 1)
        d["x"] = _randn(gen, t, h).to(dtype)  # the tokens; backward, the gradient of their output
        d["rows"] = _randn(gen, t * k, h).to(dtype)  # what the experts made of the sorted rows
        d["drows"] = _randn(gen, t * k, h).to(dtype) if c["backward"] else None  # the gradient of the sorted rows
    elif c["kind"] == "experts":
        t, k = c["tokens"], c["top_k"]
        d["ids"], _ = _picks(gen, t, c["experts"], k, 0.0)
        d["x"] = _code_rows(_activations(gen, t if c["by_token"] else t * k, c["k"]))
        d["w"] = _codes(gen, (c["experts"],), c["n"], c["k"])
        d["bias"] = 0.1 * _randn(gen, c["experts"], c["n"]) if c["bias"] else None
    else:
        t, e, h, i = c["tokens"], c["experts"], c["hidden"], c["inter"]
        d["x"] = _code_rows(_activations(gen, t, h))
        d["logits"] = _randn(gen, t, e)
        d["w"] = [_codes(gen, (e,), n, k) for n, k in ((i, h), (i, h), (h, i))]
        d["bias"] = [0.02 * _randn(gen, e, n) for n in (i, i, h)] if c["act"] == "clamped" else None
    return d


_ALPHA, _LIMIT = 1.702, 7.0

# ------------------------------------------------------------------------------ the plain forms


def _values(pair, k):
    """The values, in f32, that codes of rows stand for."""
    q, s = pair
    return (q.float().view(q.shape[0], -1, _B) * s.t()[..., None]).view(q.shape[0], -1)[:, :k]


def _weights(pair, n, k):
    """The same of matrices."""
    q, s = pair
    return q[..., :k].float() * s.repeat_interleave(_B, -2)[..., :n, :].repeat_interleave(_B, -1)[..., :k]


def _of(pair, experts):
    """The codes and scales of some experts' matrices."""
    return pair[0].view(torch.uint8)[experts].view(torch.float8_e4m3fn), pair[1][experts]


def _quantized(y):
    """The codes of rows of y, and their scales; the quotient in 64 bits, so that a code does not hang on the order of its roundings."""
    rows, k = y.shape
    p = y.new_zeros((rows, _blocks(k) * _B))
    p[:, :k] = y
    g = p.view(rows, -1, _B).double()
    a = g.abs().amax(2, keepdim=True)
    t = torch.where(a > 0, g * _TOP / a, 0.0).float()
    return t.to(torch.float8_e4m3fn).view(rows, -1), (a / _TOP).float()[..., 0].t().contiguous()


def _act(g, u, act):
    if act == "silu":
        return g / (1 + torch.exp(-g)) * u
    g, u = g.clamp(max=_LIMIT), u.clamp(-_LIMIT, _LIMIT)
    return (u + 1) * (g / (1 + torch.exp(-_ALPHA * g)))


def _plain_rows(c, d):
    x = d["x"].float()
    pair = _quantized(x if c["act"] == "none" else _act(x[:, :c["k"]], x[:, c["k"]:], c["act"]))
    return {"values": _values(pair, c["k"]).to(d["x"].dtype), "scale": pair[1]}


def _plain_matmul(c, d):
    y = _values(d["x"], c["k"]) @ _weights(d["w"], c["n"], c["k"]).t()
    return (y if d["bias"] is None else y + d["bias"]).to(_TYPES[c["dtype"]])


def _plain_sort(ids, held):
    e = ids.reshape(-1)
    e = torch.where((e >= 0) & (e < held), e, held).long()
    order = torch.argsort(e, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device="cuda")
    offsets = torch.zeros(held + 1, dtype=torch.long, device="cuda")
    offsets[1:] = torch.bincount(e, minlength=held + 1)[:held].cumsum(0)
    return e, order, place, offsets


def _plain_piles(c, d):
    t, k, h = c["tokens"], c["top_k"], c["hidden"]
    e, order, place, offsets = _plain_sort(d["ids"], d["held"])
    here, dtype = (e < d["held"])[:, None], d["x"].dtype
    rows, w = d["rows"][place].float(), d["w"].reshape(-1, 1)
    if not c["backward"]:
        sorted_rows = torch.where(here[order], d["x"][order // k], 0.0).to(dtype)
        out = torch.where(here, w * rows, 0.0).view(t, k, h).sum(1).to(dtype)
        return {"order": order.int(), "place": place.int(), "offsets": offsets.int(), "sorted": sorted_rows, "out": out}
    dx = torch.where(here, d["drows"][place].float(), 0.0).view(t, k, h).sum(1).to(dtype)
    dout = d["x"].float().repeat_interleave(k, 0)
    dy = torch.where(here, w * dout, 0.0)[order].to(dtype)
    return {"dx": dx, "dy": dy, "dw": torch.where(here, (rows * dout).sum(1, keepdim=True), 0.0).view(t, k)}


def _plain_products(x, ids, weights, bias):
    """Each row of x times its expert's matrix: the rows of every expert that has any, padded to the most that one has."""
    used, pile = torch.unique(ids, return_inverse=True)
    order = torch.argsort(pile, stable=True)
    count = torch.bincount(pile, minlength=used.numel())
    at = torch.empty_like(order)
    at[order] = torch.arange(order.numel(), device="cuda") - (count.cumsum(0) - count)[pile[order]]
    xp = x.new_zeros(used.numel(), int(count.max()), x.shape[1])
    xp[pile, at] = x
    y = torch.bmm(xp, weights(used).transpose(1, 2).contiguous())
    return (y if bias is None else y + bias[used][:, None])[pile, at]


def _plain_experts(c, d):
    k = c["top_k"]
    e, order, _, _ = _plain_sort(d["ids"], c["experts"])
    x = _values(d["x"], c["k"])
    x = x[order // k] if c["by_token"] else x
    return _plain_products(x, e[order], lambda u: _weights(_of(d["w"], u), c["n"], c["k"]), d["bias"]).to(_TYPES[c["dtype"]])


def _plain_layer(c, d):
    t, k, h, i = c["tokens"], c["top_k"], c["hidden"], c["inter"]
    ids = torch.sort(d["logits"], dim=1, descending=True, stable=True)[1][:, :k]
    p = torch.softmax(d["logits"], 1).gather(1, ids)
    w = p / p.sum(1, keepdim=True)

    def product(x, m, cols, width):
        return _plain_products(x, ids.reshape(-1), lambda u: _weights(_of(d["w"][m], u), cols, width), d["bias"] and d["bias"][m])

    x = _values(d["x"], h).repeat_interleave(k, 0)
    hidden = _values(_quantized(_act(product(x, 0, i, h), product(x, 1, i, h), c["act"])), i)
    y = product(hidden, 2, h, i).view(t, k, h)
    return {"out": (y * w[..., None]).sum(1).to(_TYPES[c["dtype"]]), "ids": ids.int(), "w": w}


_PLAIN = {"rows": _plain_rows, "matmul": _plain_matmul, "piles": _plain_piles, "experts": _plain_experts, "layer": _plain_layer}

# ------------------------------------------------------------------------------ the package's


def _own_act(act, bias=(None, None, None)):
    from coachwhip_amd import ops
    return ops.ExpertAct(gate_b=bias[0], up_b=bias[1], down_b=bias[2]) if act == "silu" else ops.ExpertAct.clamped_swiglu(_ALPHA, _LIMIT, *bias)


def _own_rows(c, d):
    from coachwhip_amd import f8
    k = c["k"]
    rows = f8.quantize_f8(d["x"]) if c["act"] == "none" else f8.swiglu_f8(d["x"][:, :k], d["x"][:, k:], _own_act(c["act"]))
    return {"values": rows.dequantize(d["x"].dtype), "scale": rows.scale}


def _own_matmul(c, d):
    from coachwhip_amd import f8
    if "product" not in d:  # built once, as when a model is loaded
        d["product"] = f8.F8MatMul(f8.F8Matrix(*d["w"], c["k"]), d["bias"])
    return d["product"].forward(f8.F8Rows(*d["x"], c["k"]), _TYPES[c["dtype"]])


def _own_piles(c, d):
    from coachwhip_amd import piles
    if not c["backward"]:
        p = piles.sort_picks(d["ids"], d["held"])
        return {"order": p.order, "place": p.place, "offsets": p.offsets, "sorted": piles.to_piles(d["x"], p),
                "out": piles.from_piles(d["rows"], d["w"], p)}
    p = piles.sort_picks(d["ids"], d["held"])
    dy, dw = piles.from_piles_grad(d["x"], d["rows"], d["w"], p)
    return {"dx": piles.to_piles_grad(d["drows"], p), "dy": dy, "dw": dw}


def _own_experts(c, d):
    from coachwhip_amd import f8, piles
    if "product" not in d:
        d["product"] = f8.F8ExpertMatMul(f8.F8ExpertBank(*d["w"], c["k"]), d["bias"])
    p = piles.sort_picks(d["ids"], c["experts"])
    return d["product"].forward(f8.F8Rows(*d["x"], c["k"]), p, _TYPES[c["dtype"]], by_token=c["by_token"])


def _own_layer(c, d):
    from coachwhip_amd import f8
    h, i = c["hidden"], c["inter"]
    if "layer" not in d:
        banks = [f8.F8ExpertBank(*w, k) for w, k in zip(d["w"], (h, h, i))]
        d["layer"] = f8.F8MoeLayer(*banks, top_k=c["top_k"], act=_own_act(c["act"], d["bias"] or (None, None, None)))
    out, ids, w = d["layer"].forward(f8.F8Rows(*d["x"], h), d["logits"], _TYPES[c["dtype"]])
    return {"out": out, "ids": ids, "w": w}


_OWN = {"rows": _own_rows, "matmul": _own_matmul, "piles": _own_piles, "experts": _own_experts, "layer": _own_layer}

# ------------------------------------------------------------------------------ a pass


def prepare(case, seed):
    return case, _inputs(case, seed)


def run(state):
    case, d = state
    if own:
        return _OWN[case["kind"]](case, d)
    return _PLAIN[case["kind"]](case, d)


def _used(experts, top_k, tokens):
    """Experts that some token picks, on average."""
    return experts * (1 - (1 - top_k / experts) ** tokens)


def work(case):
    c, b = case, _BYTES[case["dtype"]]
    if c["kind"] == "rows":
        n, halves = c["rows"] * c["k"], 1 if c["act"] == "none" else 2
        return {"bytes": n * b * (1 + halves) + 4 * c["rows"] * _blocks(c["k"]), "flops": (6 if halves == 1 else 16) * n}
    if c["kind"] == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * (k + 4 * _blocks(k)) + n * k + 4 * _blocks(n) * _blocks(k) + 4 * n * c["bias"] + b * m * n, "flops": 2 * m * n * k}
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    if c["kind"] == "piles":
        h, held = c["hidden"], t * k * (1 - c["absent"])  # the picks of experts held here
        if c["backward"]:
            return {"bytes": b * h * (2 * held + t * k + 2 * t) + 12 * t * k, "flops": 4 * held * h}
        return {"bytes": b * h * (held + t * k + 2 * t) + 16 * t * k, "flops": 2 * held * h}
    if c["kind"] == "experts":
        n, w = c["n"], c["k"]
        matrix = n * w + 4 * _blocks(n) * _blocks(w) + 4 * n * c["bias"]
        rows = t if c["by_token"] else t * k
        return {"bytes": _used(e, k, t) * matrix + rows * (w + 4 * _blocks(w)) + t * k * (4 + b * n), "flops": 2 * t * k * n * w}
    h, i = c["hidden"], c["inter"]
    expert = 3 * h * i + 12 * _blocks(h) * _blocks(i) + 4 * (2 * i + h) * (c["act"] == "clamped")
    return {"bytes": _used(e, k, t) * expert + t * (h + 4 * _blocks(h) + 4 * e + 8 * k + b * h), "flops": 6 * t * k * h * i}


# ------------------------------------------------------------------------------ the same in 64 bits


def _exact_rows(y):
    """(values, scales) of rows in codes: the quotient rounded to f32, then to three fraction bits, exponents from -6 up."""
    rows, k = y.shape
    values, scales = [], []
    for g in y.split(_B, 1):
        a = g.abs().max(dim=1, keepdim=True).values
        t = torch.where(a > 0, g * 448.0 / a, 0.0).float().double()
        step = torch.exp2(torch.clamp(torch.frexp(t).exponent - 1, min=-6) - 3.0)
        scales.append((a / 448.0).float().double())
        values.append(torch.round(t / step) * step * scales[-1])
    return torch.cat(values, 1), torch.cat(scales, 1)


def _exact_values(q, s, k):
    """Rows: s (blocks of columns, rows)."""
    return torch.cat([q[:, 128 * b:128 * (b + 1)].double() * s[b].double()[:, None] for b in range(s.shape[0])], 1)[:, :k]


def _exact_matrix(q, s, n, k):
    row, col = torch.arange(n, device="cuda") // 128, torch.arange(k, device="cuda") // 128
    return q[:, :k].double() * s.double()[row][:, col]


def _exact_hidden(g, u, act):
    if act == "silu":
        return u * g * torch.sigmoid(g)
    g, u = torch.clamp(g, max=_LIMIT), torch.clamp(u, min=-_LIMIT, max=_LIMIT)
    return (1.0 + u) * g * torch.sigmoid(g * _ALPHA)


def _exact_piles(c, d):
    t, k, held = c["tokens"], c["top_k"], d["held"]
    flat = d["ids"].reshape(-1).cpu().tolist()
    order = sorted(range(len(flat)), key=lambda p: (flat[p] if 0 <= flat[p] < held else held, p))
    order = torch.tensor(order, device="cuda")
    mine = torch.tensor([0 <= f < held for f in flat], device="cuda")
    w = torch.where(mine.view(t, k), d["w"].double(), 0.0)
    x, back = d["x"].double(), torch.empty_like(order).scatter_(0, order, torch.arange(len(flat), device="cuda")).view(t, k)
    if not c["backward"]:
        out = sum(w[:, j, None] * d["rows"][back[:, j]].double() for j in range(k))
        return {"order": None, "place": None, "offsets": None, "sorted": x[torch.div(order, k, rounding_mode="floor")] * mine[order][:, None], "out": out}
    m = mine.view(t, k)
    dx = sum(m[:, j, None] * d["drows"][back[:, j]].double() for j in range(k))
    dw = torch.stack([m[:, j] * (x * d["rows"][back[:, j]].double()).sum(1) for j in range(k)], 1)
    dy = torch.empty(t * k, c["hidden"], dtype=torch.float64, device="cuda")
    for j in range(k):
        dy[back[:, j]] = w[:, j, None] * x
    return {"dx": dx, "dy": dy, "dw": dw}


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "rows":
        y = d["x"].double()
        values, scale = _exact_rows(y if c["act"] == "none" else _exact_hidden(y[:, :c["k"]], y[:, c["k"]:], c["act"]))
        return {"values": values, "scale": scale.t().contiguous()}
    if c["kind"] == "matmul":
        y = _exact_values(*d["x"], c["k"]) @ _exact_matrix(*d["w"], c["n"], c["k"]).t()
        return y if d["bias"] is None else y + d["bias"].double()
    if c["kind"] == "piles":
        return _exact_piles(c, d)
    if c["kind"] == "experts":
        k, flat = c["top_k"], d["ids"].reshape(-1)
        x = _exact_values(*d["x"], c["k"])
        parts, at = [], 0
        for e in range(c["experts"]):  # an expert's picks follow one another, in the order of the tokens
            p = torch.nonzero(flat == e)[:, 0]
            if p.numel():
                rows = x[p // k] if c["by_token"] else x[at:at + p.numel()]
                y = rows @ _exact_matrix(d["w"][0][e], d["w"][1][e], c["n"], c["k"]).t()
                parts.append(y if d["bias"] is None else y + d["bias"][e].double())
                at += p.numel()
        return torch.cat(parts)
    h, i = c["hidden"], c["inter"]
    best, ids = torch.sort(d["logits"].double(), dim=1, descending=True, stable=True)
    ids, w = ids[:, :c["top_k"]], torch.softmax(best[:, :c["top_k"]], 1)  # over the picks alone: the others' terms cancel
    x = _exact_values(*d["x"], h)
    out = torch.zeros(c["tokens"], h, dtype=torch.float64, device="cuda")
    for e in torch.unique(ids).tolist():
        t, j = torch.nonzero(ids == e, as_tuple=True)
        b = [0.0] * 3 if d["bias"] is None else [v[e].double() for v in d["bias"]]
        g, u = (x[t] @ _exact_matrix(d["w"][m][0][e], d["w"][m][1][e], i, h).t() + b[m] for m in (0, 1))
        hid = _exact_rows(_exact_hidden(g, u, c["act"]))[0]
        out.index_add_(0, t, w[t, j][:, None] * (hid @ _exact_matrix(d["w"][2][0][e], d["w"][2][1][e], h, i).t() + b[2]))
    return {"out": out, "ids": None, "w": w}
