"""What the 8-bit float entry points and the piles refuse, on the host: nothing here reaches a device."""
import ctypes

import pytest
import torch

import coachwhip_amd as cw
from coachwhip_amd import f8, piles
from coachwhip_amd import formats as F
from coachwhip_amd._lib import CW_EINVAL, CW_ENOTSUP, CW_F8_MAX_K, CW_OK, F8MoeDesc

P, Q = ctypes.c_void_p(4096), ctypes.c_void_p(4097)  # aligned, unaligned; never read


def test_row_bytes():
    L = cw.lib()
    assert [L.cw_f8_row_bytes(k) for k in (-1, 0, 1, 128, 129, 2880)] == [0, 0, 128, 128, 256, 2944]
    assert all(L.cw_f8_row_bytes(k) == f8.row_bytes(k) == 128 * f8.blocks(k) for k in range(1, 400))


def quantize(dtype=F.F32, x=P, ldx=64, rows=2, k=64, q=P, scale=P):
    return cw.lib().cw_quantize_f8(dtype, x, ldx, rows, k, q, scale, None)


def matrix(dtype=F.F32, x=P, ldx=64, rows=2, k=64, q=P, scale=P):
    return cw.lib().cw_quantize_f8_matrix(dtype, x, ldx, rows, k, q, scale, None)


def swiglu(dtype=F.BF16, g=P, u=P, ld=64, rows=2, k=64, act=0, q=P, scale=P):
    return cw.lib().cw_swiglu_f8(dtype, g, u, ld, rows, k, act, 1.0, 7.0, q, scale, None)


def dequantize(q=P, scale=P, rows=2, k=64, dtype=F.F32, out=P):
    return cw.lib().cw_dequantize_f8(q, scale, rows, k, dtype, out, None)


def matmul(w=P, ws=P, n=8, k=64, x=P, xs=P, m=2, bias=None, dtype=F.F32, y=P, ldy=8):
    return cw.lib().cw_f8_matmul(w, ws, n, k, x, xs, m, bias, dtype, y, ldy, None)


def experts(w=P, stride=1024, ws=P, E=4, n=8, k=64, x=P, xs=P, m=2, order=P, K=3, picks=6, tiles=P, bias=None, dtype=F.F32, y=P, ldy=8):
    return cw.lib().cw_f8_matmul_experts(w, stride, ws, E, n, k, x, xs, m, order, K, picks, tiles, bias, dtype, y, ldy, None)


ROWS = [({"dtype": F.Q8_0}, CW_ENOTSUP), ({"rows": -1}, CW_EINVAL), ({"rows": 1 << 31}, CW_EINVAL), ({"k": 0}, CW_EINVAL),
        ({"k": CW_F8_MAX_K + 1}, CW_ENOTSUP), ({"rows": 1 << 27}, CW_ENOTSUP), ({"q": None}, CW_EINVAL), ({"q": Q}, CW_EINVAL), ({"scale": None}, CW_EINVAL)]
PRODUCT = [({"n": 0}, CW_EINVAL), ({"k": 0}, CW_EINVAL), ({"m": -1}, CW_EINVAL), ({"m": 1 << 31}, CW_EINVAL), ({"n": 1 << 31, "ldy": 1 << 32}, CW_EINVAL),
           ({"k": CW_F8_MAX_K + 1}, CW_ENOTSUP), ({"ldy": 7}, CW_EINVAL), ({"dtype": F.Q4_K}, CW_ENOTSUP), ({"w": None}, CW_EINVAL), ({"ws": None}, CW_EINVAL),
           ({"x": None}, CW_EINVAL), ({"xs": None}, CW_EINVAL), ({"y": None}, CW_EINVAL), ({"w": Q}, CW_EINVAL), ({"x": Q}, CW_EINVAL)]


@pytest.mark.parametrize("call,bad,status", [(c, b, s) for c in (quantize, matrix, swiglu, dequantize) for b, s in ROWS]
                         + [(c, b, s) for c in (matmul, experts) for b, s in PRODUCT] + [
    (quantize, {"x": None}, CW_EINVAL), (quantize, {"ldx": 63}, CW_EINVAL), (matrix, {"x": None}, CW_EINVAL), (matrix, {"ldx": 63}, CW_EINVAL),
    (swiglu, {"g": None}, CW_EINVAL), (swiglu, {"u": None}, CW_EINVAL), (swiglu, {"ld": 63}, CW_EINVAL), (swiglu, {"act": 2}, CW_EINVAL),
    (dequantize, {"out": None}, CW_EINVAL), (matmul, {"n": 1 << 27, "ldy": 1 << 27}, CW_ENOTSUP),
    (experts, {"stride": 1008}, CW_EINVAL), (experts, {"stride": 1032}, CW_EINVAL), (experts, {"E": 0}, CW_EINVAL), (experts, {"E": 1025}, CW_EINVAL),
    (experts, {"K": 0}, CW_EINVAL), (experts, {"picks": 7}, CW_EINVAL), (experts, {"order": None}, CW_EINVAL), (experts, {"tiles": None}, CW_EINVAL),
    (experts, {"tiles": Q}, CW_EINVAL), (experts, {"picks": 1 << 28}, CW_EINVAL),
    (experts, {"n": 1 << 26, "ldy": 1 << 26, "stride": 1 << 33, "m": 1000, "picks": 3000}, CW_ENOTSUP)])
def test_rows_and_products_refuse(call, bad, status):
    assert call(**bad) == status and cw.lib().cw_last_error()


def test_no_rows_are_no_call():
    assert quantize(rows=0, x=None, q=None, scale=None) == matrix(rows=0, x=None, q=None, scale=None) == CW_OK
    assert swiglu(rows=0, g=None, u=None, q=None, scale=None) == dequantize(rows=0, q=None, scale=None, out=None) == CW_OK
    assert matmul(m=0, x=None, xs=None, y=None) == experts(m=0, picks=0, x=None, xs=None, y=None, tiles=None) == CW_OK


def sort(ids=P, picks=6, E=4, order=P, place=P, offsets=P, tiles=P, ws=None, ws_bytes=0):
    return cw.lib().cw_sort_picks(ids, picks, E, order, place, offsets, tiles, ws, ws_bytes, None)


def to_piles(dtype=F.BF16, x=P, ldx=64, T=2, K=3, E=4, h=64, place=P, offsets=P, rows=P):  # (its place is the order)
    return cw.lib().cw_to_piles(dtype, x, ldx, T, K, E, h, place, offsets, rows, None)


def from_piles(dtype=F.BF16, rows=P, ldx=64, w=None, T=2, K=3, E=4, h=64, place=P, offsets=P, out=P):
    return cw.lib().cw_from_piles(dtype, rows, ldx, w, T, K, E, h, place, offsets, out, None)


def from_piles_grad(dtype=F.BF16, dout=P, ldx=64, rows=P, ldr=64, w=P, T=2, K=3, E=4, h=64, place=P, offsets=P, drows=P, dw=P):
    return cw.lib().cw_from_piles_grad(dtype, dout, ldx, rows, ldr, w, T, K, E, h, place, offsets, drows, dw, None)


WAY = [({"dtype": F.Q8_0}, CW_ENOTSUP), ({"T": -1}, CW_EINVAL), ({"K": 0}, CW_EINVAL), ({"E": 0}, CW_EINVAL), ({"E": 1025}, CW_EINVAL), ({"h": 0}, CW_EINVAL),
       ({"h": 1 << 31}, CW_EINVAL), ({"ldx": 63}, CW_EINVAL), ({"place": None}, CW_EINVAL), ({"offsets": None}, CW_EINVAL), ({"T": 1 << 27, "K": 2}, CW_ENOTSUP)]


@pytest.mark.parametrize("call,bad,status", [(c, b, s) for c in (to_piles, from_piles, from_piles_grad) for b, s in WAY] + [
    (to_piles, {"x": None}, CW_EINVAL), (to_piles, {"rows": None}, CW_EINVAL), (from_piles, {"rows": None}, CW_EINVAL), (from_piles, {"out": None}, CW_EINVAL),
    (from_piles_grad, {"dout": None}, CW_EINVAL), (from_piles_grad, {"rows": None}, CW_EINVAL), (from_piles_grad, {"w": None}, CW_EINVAL),
    (from_piles_grad, {"drows": None}, CW_EINVAL), (from_piles_grad, {"dw": None}, CW_EINVAL), (from_piles_grad, {"ldr": 63}, CW_EINVAL),
    (sort, {"E": 0}, CW_EINVAL), (sort, {"E": 1025}, CW_EINVAL), (sort, {"picks": -1}, CW_EINVAL), (sort, {"picks": 1 << 28}, CW_ENOTSUP), (sort, {"ids": None}, CW_EINVAL),
    (sort, {"order": None}, CW_EINVAL), (sort, {"place": None}, CW_EINVAL), (sort, {"offsets": None}, CW_EINVAL), (sort, {"tiles": None}, CW_EINVAL),
    (sort, {"tiles": Q}, CW_EINVAL), (sort, {"picks": 1 << 20}, CW_EINVAL), (sort, {"picks": 1 << 20, "ws": P, "ws_bytes": 100}, CW_EINVAL)])
def test_piles_refuse(call, bad, status):
    assert call(**bad) == status and cw.lib().cw_last_error()


def test_no_tokens_are_no_call():
    assert to_piles(T=0, x=None, place=None, rows=None) == from_piles(T=0, rows=None, out=None) == from_piles_grad(T=0, dout=None, dw=None) == CW_OK


def test_sizes_of_the_sort():
    L = cw.lib()
    assert L.cw_pile_tiles_bytes(-1, 4) == L.cw_pile_tiles_bytes(4, 0) == 0 and L.cw_pile_tiles_bytes(0, 4) >= 16
    assert L.cw_sort_picks_workspace_size(2048, 256) == 0 < L.cw_sort_picks_workspace_size(2049, 256)


def desc(**kw):
    d = F8MoeDesc()
    d.n_experts, d.top_k, d.hidden, d.inter, d.norm, d.act, d.alpha, d.limit = 8, 2, 100, 36, 1, 0, 1.0, 7.0
    for m, (n, k) in enumerate(((36, 100), (36, 100), (100, 36))):
        d.w[m], d.scale[m], d.slot_stride[m] = 4096, 4096, n * f8.row_bytes(k)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def layer(d, T=2, x=P, xs=P, logits=P, dtype=F.F32, out=P, ws=P, ws_bytes=1 << 40):
    return cw.lib().cw_f8_moe_layer(ctypes.byref(d), x, xs, logits, T, dtype, out, None, None, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    ({"n_experts": 0}, CW_EINVAL), ({"n_experts": 1025}, CW_EINVAL), ({"top_k": 0}, CW_EINVAL), ({"top_k": 9}, CW_EINVAL), ({"top_k": 33, "n_experts": 64}, CW_EINVAL),
    ({"hidden": 0}, CW_EINVAL), ({"inter": 0}, CW_EINVAL), ({"hidden": CW_F8_MAX_K + 1}, CW_ENOTSUP), ({"inter": CW_F8_MAX_K + 1}, CW_ENOTSUP), ({"act": 2}, CW_EINVAL)])
def test_layer_descriptors_refuse(kw, status):
    d = desc(**kw)
    assert layer(d) == status and cw.lib().cw_f8_moe_workspace_size(ctypes.byref(d), 2) == 0


@pytest.mark.parametrize("what,m,value", [("w", 0, None), ("w", 2, 4097), ("scale", 1, None), ("slot_stride", 0, 36 * 128 - 16), ("slot_stride", 2, 100 * 128 + 8)])
def test_layer_matrices_refuse(what, m, value):
    d = desc()
    getattr(d, what)[m] = value
    assert layer(d) == CW_EINVAL


@pytest.mark.parametrize("kw,status", [({"T": -1}, CW_EINVAL), ({"T": 1 << 27}, CW_ENOTSUP), ({"x": None}, CW_EINVAL), ({"x": Q}, CW_EINVAL), ({"xs": None}, CW_EINVAL),
                                       ({"logits": None}, CW_EINVAL), ({"out": None}, CW_EINVAL), ({"dtype": F.Q8_0}, CW_ENOTSUP), ({"ws": None}, CW_EINVAL),
                                       ({"ws": Q}, CW_EINVAL), ({"ws_bytes": 100}, CW_EINVAL)])
def test_layer_calls_refuse(kw, status):
    assert layer(desc(), **kw) == status
    assert layer(desc(), T=0, x=None, logits=None, out=None, ws=None) == CW_OK


def test_python_refuses_tensors_of_the_host():
    x = torch.zeros(2, 128)
    for call in (lambda: f8.quantize_f8(x), lambda: f8.swiglu_f8(x, x), lambda: f8.F8Rows(x.to(torch.float8_e4m3fn), torch.zeros(1, 2), 128),
                 lambda: f8.F8Matrix.from_float(x), lambda: piles.sort_picks(torch.zeros(2, 2, dtype=torch.int32), 4)):
        with pytest.raises(cw.CwError):
            call()
