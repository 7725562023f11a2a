"""What the 8-bit integer entry points refuse, on the host: nothing here reaches a device."""
import ctypes

import pytest
import torch

import coachwhip_amd as cw
from coachwhip_amd import formats as F
from coachwhip_amd import i8
from coachwhip_amd._lib import CW_EINVAL, CW_ENOTSUP, CW_I8_MAX_K, CW_OK, I8MoeDesc

P, Q = ctypes.c_void_p(4096), ctypes.c_void_p(4097)  # aligned, unaligned; never read


def test_row_bytes():
    L = cw.lib()
    assert [L.cw_i8_row_bytes(k) for k in (-1, 0, 1, 128, 129, 2880)] == [0, 0, 128, 128, 256, 2944]
    assert all(L.cw_i8_row_bytes(k) == i8.row_bytes(k) for k in range(1, 400))


def quantize(dtype=F.F32, x=P, ldx=64, rows=2, k=64, q=P, scale=P):
    return cw.lib().cw_quantize_i8(dtype, x, ldx, rows, k, q, scale, None)


def swiglu(dtype=F.BF16, g=P, u=P, ld=64, rows=2, k=64, act=0, q=P, scale=P):
    return cw.lib().cw_swiglu_i8(dtype, g, u, ld, rows, k, act, 1.0, 7.0, q, scale, None)


def norm(dtype=F.F16, x=P, ldx=64, r=P, ldr=64, w=P, eps=1e-6, rows=2, k=64, total=P, y=None, q=P, scale=P):
    return cw.lib().cw_rmsnorm_i8(dtype, x, ldx, r, ldr, w, eps, rows, k, total, y, q, scale, None)


def dequantize(q=P, scale=P, rows=2, k=64, dtype=F.F32, out=P):
    return cw.lib().cw_dequantize_i8(q, scale, rows, k, dtype, out, None)


def matmul(w=P, ws=P, n=8, k=64, x=P, xs=P, m=2, bias=None, dtype=F.F32, y=P, ldy=8):
    return cw.lib().cw_i8_matmul(w, ws, n, k, x, xs, m, bias, dtype, y, ldy, None)


ROWS = [({"dtype": F.Q8_0}, CW_ENOTSUP), ({"rows": -1}, CW_EINVAL), ({"rows": 1 << 31}, CW_EINVAL), ({"k": 0}, CW_EINVAL),
        ({"k": CW_I8_MAX_K + 1}, CW_ENOTSUP), ({"q": None}, CW_EINVAL), ({"q": Q}, CW_EINVAL), ({"scale": None}, CW_EINVAL)]


@pytest.mark.parametrize("call,bad,status", [(c, b, s) for c in (quantize, swiglu, norm, dequantize) for b, s in ROWS] + [
    (quantize, {"x": None}, CW_EINVAL), (quantize, {"ldx": 63}, CW_EINVAL),
    (swiglu, {"g": None}, CW_EINVAL), (swiglu, {"u": None}, CW_EINVAL), (swiglu, {"ld": 63}, CW_EINVAL), (swiglu, {"act": 2}, CW_EINVAL),
    (norm, {"x": None}, CW_EINVAL), (norm, {"w": None}, CW_EINVAL), (norm, {"ldx": 63}, CW_EINVAL), (norm, {"ldr": 63}, CW_EINVAL),
    (norm, {"eps": -1e-6}, CW_EINVAL), (norm, {"eps": float("nan")}, CW_EINVAL), (norm, {"r": None}, CW_EINVAL),
    (dequantize, {"out": None}, CW_EINVAL),
    (matmul, {"n": 0}, CW_EINVAL), (matmul, {"k": 0}, CW_EINVAL), (matmul, {"m": -1}, CW_EINVAL), (matmul, {"m": 1 << 31}, CW_EINVAL),
    (matmul, {"n": 1 << 31, "ldy": 1 << 32}, CW_EINVAL), (matmul, {"k": CW_I8_MAX_K + 1}, CW_ENOTSUP), (matmul, {"ldy": 7}, CW_EINVAL),
    (matmul, {"dtype": F.Q4_K}, CW_ENOTSUP), (matmul, {"w": None}, CW_EINVAL), (matmul, {"ws": None}, CW_EINVAL), (matmul, {"x": None}, CW_EINVAL),
    (matmul, {"xs": None}, CW_EINVAL), (matmul, {"y": None}, CW_EINVAL), (matmul, {"w": Q}, CW_EINVAL), (matmul, {"x": Q}, CW_EINVAL)])
def test_rows_and_products_refuse(call, bad, status):
    assert call(**bad) == status and cw.lib().cw_last_error()


def test_no_rows_are_no_call():
    assert quantize(rows=0, x=None, q=None, scale=None) == swiglu(rows=0, g=None, u=None, q=None, scale=None) == CW_OK
    assert norm(rows=0, x=None, r=None, w=None, total=None, q=None, scale=None) == dequantize(rows=0, q=None, scale=None, out=None) == CW_OK
    assert matmul(m=0, x=None, xs=None, y=None) == CW_OK


def desc(**kw):
    d = I8MoeDesc()
    d.n_experts, d.top_k, d.hidden, d.inter, d.norm, d.act, d.alpha, d.limit = 8, 2, 100, 36, 1, 0, 1.0, 7.0
    for m, (n, k) in enumerate(((36, 100), (36, 100), (100, 36))):
        d.w[m], d.scale[m], d.slot_stride[m] = 4096, 4096, n * i8.row_bytes(k)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def layer(d, T=2, x=P, xs=P, logits=P, dtype=F.F32, out=P, ws=P, ws_bytes=1 << 40):
    return cw.lib().cw_i8_moe_layer(ctypes.byref(d), x, xs, logits, T, dtype, out, None, None, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    ({"n_experts": 0}, CW_EINVAL), ({"n_experts": 1025}, CW_EINVAL), ({"top_k": 0}, CW_EINVAL), ({"top_k": 9}, CW_EINVAL), ({"top_k": 33, "n_experts": 64}, CW_EINVAL),
    ({"hidden": 0}, CW_EINVAL), ({"inter": -1}, CW_EINVAL), ({"hidden": CW_I8_MAX_K + 1}, CW_ENOTSUP), ({"inter": CW_I8_MAX_K + 1}, CW_ENOTSUP),
    ({"act": 2}, CW_EINVAL), ({"hidden": 200}, CW_EINVAL)])  # (the last: strides below the matrices)
def test_layer_refuses_bad_descriptors(kw, status):
    d = desc(**kw)
    assert layer(d) == status and cw.lib().cw_i8_moe_workspace_size(ctypes.byref(d), 2) == 0


def test_layer_refuses_bad_calls():
    for m in range(3):
        for field, v in (("w", None), ("scale", None), ("w", 4097), ("slot_stride", 0), ("slot_stride", (1 << 20) + 8)):
            d = desc()
            getattr(d, field)[m] = v
            assert layer(d) == CW_EINVAL, (m, field, v)
    d = desc()
    assert layer(d, T=-1) == CW_EINVAL and layer(d, T=1 << 27) == CW_ENOTSUP
    assert layer(d, dtype=F.MXFP4) == CW_ENOTSUP
    for bad in ({"x": None}, {"x": Q}, {"xs": None}, {"logits": None}, {"out": None}, {"ws": None}, {"ws": Q}):
        assert layer(d, **bad) == CW_EINVAL, bad
    need = cw.lib().cw_i8_moe_workspace_size(ctypes.byref(d), 2)
    assert need > 0 and layer(d, ws_bytes=need - 1) == CW_EINVAL
    assert cw.lib().cw_i8_moe_layer(None, P, P, P, 1, F.F32, P, None, None, P, 1 << 40, None) == CW_EINVAL
    assert layer(d, T=0, x=None, xs=None, logits=None, out=None, ws=None, ws_bytes=0) == CW_OK


def test_layer_workspace_grows_with_its_tokens():
    d, last = desc(n_experts=256, top_k=8), 0
    for t in [*range(1, 70), 100, 1000, 5000]:
        need = cw.lib().cw_i8_moe_workspace_size(ctypes.byref(d), t)
        assert need >= last
        last = need


def test_host_tensors_are_refused():
    x, v = torch.zeros(2, 128), torch.zeros(128)
    for call in (lambda: i8.quantize_i8(x), lambda: i8.swiglu_i8(x, x), lambda: i8.rmsnorm_i8(x, v, 1e-6), lambda: i8.I8Rows(x.to(torch.int8), v[:2], 128),
                 lambda: i8.I8Matrix(x.to(torch.int8), v[:2], 128), lambda: i8.I8ExpertBank(x.to(torch.int8)[None], v[None, :2], 128)):
        with pytest.raises(cw.CwError):
            call()
