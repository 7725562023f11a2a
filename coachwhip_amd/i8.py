"""The 8-bit integer path of a MoE block: weights with a scale per output channel, activations with a
scale per token, products summed exactly in 32-bit integers.

- ``rmsnorm_i8``: the residual's addition and an RMS norm, its rows as codes;
- ``quantize_i8`` / ``swiglu_i8``: rows of floats, or of a SwiGLU, as codes;
- ``I8MatMul``: codes times an ``I8Matrix``, beside ``ops.QMatMul``;
- ``I8MoeLayer``: a layer of 8-bit experts, beside ``ops.MoeLayer``.

``I8Matrix.from_qtensor`` and ``I8ExpertBank.from_bank`` lay GGUF weights out once, when a model is
loaded. No counterpart in the reference, whose activations are floats. Activations are f32, f16 or
bf16 tensors, on the current stream of their own device; all arithmetic runs in libcwmoe.so. Shape and type errors raise
``CwError``.
"""
import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import formats as F
from . import ops
from ._lib import CW_EINVAL, CW_I8_MAX_K, CwError, I8MoeDesc, check, lib

_DTYPES = {torch.float32: F.F32, torch.float16: F.F16, torch.bfloat16: F.BF16}
_SILU = ops.ExpertAct.silu()


def row_bytes(k: int) -> int:
    """Bytes of a row of k codes: whole 128 bytes, zeros past k."""
    return (k + 127) // 128 * 128


def _fail(msg, *a):
    raise CwError(CW_EINVAL, msg % a)


def _same_device(first, *others):
    d = first.device
    for t in others:
        if t is not None and t.device != d:
            _fail("tensors on %s and %s", d, t.device)


def _elsewhere(t):
    """Whether the tensor's device is not the current one, to which a launch would go."""
    return t.device.index != torch.cuda.current_device()


def _stream(t):
    """The current stream of the tensor's device (without the Stream object that torch.cuda.current_stream makes, 3 of
    a small call's 11 us)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _floats(t, what):
    """A device tensor of rows of floats whose elements are adjacent; the elements from a row to the next."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _DTYPES:
        _fail("%s must be an f32, f16 or bf16 device tensor", what)
    shape = t.shape
    if len(shape) != 2 or shape[1] == 0:
        _fail("%s must be rows of values, got %s", what, tuple(shape))
    ld, one = t.stride()
    if one != 1 and shape[1] > 1:
        _fail("%s: rows of adjacent elements, got strides %s", what, t.stride())
    if shape[0] <= 1:
        return shape[1]
    if ld < shape[1]:
        _fail("%s: rows %d elements apart overlap", what, ld)
    return ld


def _vector(t, n, what):
    if t is not None:
        ops._need(t, torch.float32, what)
        if t.numel() != n:
            _fail("%s of %d values, expected %d", what, t.numel(), n)


def _codes(q, scale, k, lead, what):
    if not isinstance(q, torch.Tensor) or not isinstance(scale, torch.Tensor) or not q.is_cuda or q.dtype != torch.int8 or scale.dtype != torch.float32:
        _fail("%s: int8 codes and f32 scales on a device", what)
    if q.device != scale.device or not q.is_contiguous() or not scale.is_contiguous():
        _fail("%s: contiguous codes and scales on one device", what)
    shape = q.shape
    if len(shape) != lead + 1 or k <= 0 or shape[-1] != row_bytes(k):
        _fail("%s codes %s: rows of %d bytes for %d codes", what, tuple(shape), row_bytes(k), k)
    if scale.shape != shape[:-1]:
        _fail("%s scales %s for codes %s", what, tuple(scale.shape), tuple(shape))
    if q.data_ptr() % 16:
        _fail("%s codes must be 16-byte aligned", what)


@dataclass
class I8Rows:
    """Rows of k codes: ``q`` (rows, row_bytes(k)) int8, zeros past k, and ``scale`` (rows,) f32."""
    q: torch.Tensor
    scale: torch.Tensor
    k: int

    def __post_init__(self):
        _codes(self.q, self.scale, self.k, 1, "rows")

    def __len__(self):
        return self.q.shape[0]

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """(rows, k) of code * scale."""
        if dtype not in _DTYPES:
            _fail("dequantize to %s", dtype)
        q = self.q
        if _elsewhere(q):
            with torch.cuda.device(q.device):
                return self.dequantize(dtype)
        rows = q.shape[0]
        out = q.new_empty((rows, self.k), dtype=dtype)
        check(lib().cw_dequantize_i8(q.data_ptr(), self.scale.data_ptr(), rows, self.k, _DTYPES[dtype], out.data_ptr(), _stream(q)))
        return out


def _new_rows(x, rows, k):
    if k > CW_I8_MAX_K:
        _fail("rows of %d codes above %d", k, CW_I8_MAX_K)
    r = object.__new__(I8Rows)
    r.q, r.scale, r.k = x.new_empty((rows, row_bytes(k)), dtype=torch.int8), x.new_empty(rows, dtype=torch.float32), k
    return r


def quantize_i8(x: torch.Tensor) -> I8Rows:
    """Rows (any stride between them) as codes: scale = max|x| / 127, code = x / scale to the nearest."""
    ld = _floats(x, "x")
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return quantize_i8(x)
    rows, k = x.shape
    r = _new_rows(x, rows, k)
    check(lib().cw_quantize_i8(_DTYPES[x.dtype], x.data_ptr(), ld, rows, k, r.q.data_ptr(), r.scale.data_ptr(), _stream(x)))
    return r


def swiglu_i8(g: torch.Tensor, u: torch.Tensor, act: Optional[ops.ExpertAct] = None) -> I8Rows:
    """silu(g) * u, or the clamped SwiGLU of ``act``, as codes. g and u: rows of one type and stride (the
    halves of one product's rows). Biases belong to the product (``I8MatMul``): ``act`` must have none."""
    act = act or _SILU
    if act.gate_b is not None or act.up_b is not None or act.down_b is not None or act.pad:
        _fail("swiglu_i8: an activation with biases or padding")
    ld = _floats(g, "gate")
    if _floats(u, "up") != ld or u.dtype != g.dtype or u.shape != g.shape:
        _fail("gate %s %s and up %s %s differ in shape, type or stride", tuple(g.shape), g.dtype, tuple(u.shape), u.dtype)
    _same_device(g, u)
    if _elsewhere(g):
        with torch.cuda.device(g.device):
            return swiglu_i8(g, u, act)
    rows, k = g.shape
    r = _new_rows(g, rows, k)
    check(lib().cw_swiglu_i8(_DTYPES[g.dtype], g.data_ptr(), u.data_ptr(), ld, rows, k, act.kind, act.alpha, act.limit, r.q.data_ptr(),
                             r.scale.data_ptr(), _stream(g)))
    return r


def rmsnorm_i8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None, keep_y: bool = False):
    """(rows as codes, the sum or None, y or None): h = x + residual in x's type (returned as the sum when a
    residual is given), y = h * weight / sqrt(mean(h^2) + eps) as codes, and as f32 rows with ``keep_y``
    (``ops.router_logits`` reads them)."""
    ldx = _floats(x, "x")
    rows, k = x.shape
    if weight is None:
        _fail("rmsnorm_i8: a weight of %d values", k)
    _vector(weight, k, "weight")
    ldr, total, y = 0, None, None
    if residual is not None:
        ldr = _floats(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype:
            _fail("residual %s %s for x %s %s", tuple(residual.shape), residual.dtype, tuple(x.shape), x.dtype)
    _same_device(x, weight, residual)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return rmsnorm_i8(x, weight, eps, residual, keep_y)
    r = _new_rows(x, rows, k)
    if residual is not None:
        total = x.new_empty((rows, k))
    if keep_y:
        y = x.new_empty((rows, k), dtype=torch.float32)
    check(lib().cw_rmsnorm_i8(_DTYPES[x.dtype], x.data_ptr(), ldx, _ptr(residual), ldr, weight.data_ptr(), eps, rows, k, _ptr(total), _ptr(y),
                              r.q.data_ptr(), r.scale.data_ptr(), _stream(x)))
    return r, total, y


@dataclass
class I8Matrix:
    """An (n, k) weight: ``q`` (n, row_bytes(k)) int8 and ``scale`` (n,) f32, one per output channel."""
    q: torch.Tensor
    scale: torch.Tensor
    k: int

    def __post_init__(self):
        _codes(self.q, self.scale, self.k, 1, "matrix")

    @property
    def shape(self):
        return self.q.shape[0], self.k

    @classmethod
    def from_float(cls, w: torch.Tensor):
        r = quantize_i8(w)
        return cls(r.q, r.scale, r.k)

    @classmethod
    def from_qtensor(cls, w: ops.QTensor):
        with torch.cuda.device(w.data.device):
            return cls.from_float(w.dequantize())


class I8MatMul:
    """y = x . W^T (+ bias) for 8-bit rows x and an 8-bit W: each output one exact integer sum, scaled."""

    def __init__(self, matrix: I8Matrix, bias: Optional[torch.Tensor] = None):
        _vector(bias, matrix.shape[0], "bias")
        _same_device(matrix.q, bias)
        self.w, self.bias = matrix, bias

    def forward(self, xs: I8Rows, dtype=torch.float32) -> torch.Tensor:
        w, q, k = self.w.q, xs.q, xs.k
        if k != self.w.k:
            _fail("rows of %d incompatible with %s", k, self.w.shape)
        if dtype not in _DTYPES:
            _fail("i8 matmul to %s", dtype)
        _same_device(w, q)
        if _elsewhere(q):
            with torch.cuda.device(q.device):
                return self.forward(xs, dtype)
        m, n = q.shape[0], w.shape[0]
        y = q.new_empty((m, n), dtype=dtype)
        check(lib().cw_i8_matmul(w.data_ptr(), self.w.scale.data_ptr(), n, k, q.data_ptr(), xs.scale.data_ptr(), m, _ptr(self.bias),
                                 _DTYPES[dtype], y.data_ptr(), n, _stream(q)))
        return y

    __call__ = forward


@dataclass
class I8ExpertBank:
    """One matrix of every expert: ``q`` (experts, n, row_bytes(k)) int8, ``scale`` (experts, n) f32."""
    q: torch.Tensor
    scale: torch.Tensor
    k: int

    def __post_init__(self):
        _codes(self.q, self.scale, self.k, 2, "bank")

    @property
    def n(self):
        return self.q.shape[1]

    @classmethod
    def from_float(cls, w: torch.Tensor):
        """Of (experts, n, k) floats."""
        if w.dim() != 3:
            _fail("bank: (experts, n, k) weights, got %s", tuple(w.shape))
        e, n, k = w.shape
        r = quantize_i8(w.reshape(e * n, k))
        return cls(r.q.view(e, n, -1), r.scale.view(e, n), k)

    @classmethod
    def from_bank(cls, bank: ops.ExpertBank):
        """Of a bank of GGUF blocks, one expert's floats at a time."""
        n, k, e = bank.n, bank.k, bank.n_slots
        q = torch.empty((e, n, row_bytes(k)), dtype=torch.int8, device=bank.data.device)
        scale = torch.empty((e, n), dtype=torch.float32, device=bank.data.device)
        size = F.matrix_bytes(bank.dtype, n, k)
        with torch.cuda.device(bank.data.device):
            for s in range(e):
                raw = bank.data[s * bank.slot_stride:s * bank.slot_stride + size]
                r = quantize_i8(ops.dequantize(bank.dtype, raw, n * k).view(n, k))
                q[s], scale[s] = r.q, r.scale
        return cls(q, scale, k)


class I8MoeLayer:
    """A MoE layer of 8-bit experts, all resident: ``ops.MoeLayer`` on 8-bit rows."""

    def __init__(self, gate: I8ExpertBank, up: I8ExpertBank, down: I8ExpertBank, top_k: int, norm_topk_prob: bool = True,
                 act: Optional[ops.ExpertAct] = None):
        act = act or ops.ExpertAct.silu()
        e, inter, hidden = gate.q.shape[0], gate.n, gate.k
        for b, n, k, what in ((up, inter, hidden, "up"), (down, hidden, inter, "down")):
            if b.q.shape[0] != e or b.n != n or b.k != k:
                _fail("%s bank of %d (%d, %d) for %d experts (%d, %d)", what, b.q.shape[0], b.n, b.k, e, n, k)
        if act.pad not in (0, inter):
            _fail("i8 moe: padding (rows of codes are padded by themselves)")
        biases = (act.gate_b, act.up_b, act.down_b)
        for b, n, what in zip(biases, (inter, inter, hidden), ("gate", "up", "down")):
            _vector(b, e * n, "%s bias" % what)
        _same_device(gate.q, up.q, down.q, *biases)
        self.banks, self.act = (gate, up, down), act
        self.n_experts, self.top_k, self.hidden, self.inter = e, top_k, hidden, inter
        d = I8MoeDesc()
        d.n_experts, d.top_k, d.hidden, d.inter, d.norm = e, top_k, hidden, inter, int(norm_topk_prob)
        d.act, d.alpha, d.limit = act.kind, act.alpha, act.limit
        for m, b in enumerate(self.banks):
            d.w[m], d.scale[m], d.slot_stride[m] = b.q.data_ptr(), b.scale.data_ptr(), b.q.stride(0)
            d.bias[m] = None if biases[m] is None else biases[m].data_ptr()
        self.desc = d

    def forward(self, xs: I8Rows, logits: torch.Tensor, dtype=torch.float32):
        """xs T rows of hidden, logits (T, E) f32 -> (out (T, hidden), ids (T, K), w (T, K)). The workspace is
        allocated for the call (on the stream, or in the graph that captures it)."""
        ops._need(logits, torch.float32, "logits")
        t = len(xs)
        if xs.k != self.hidden or logits.shape != (t, self.n_experts):
            _fail("rows of %d / logits %s do not fit the layer", xs.k, tuple(logits.shape))
        if dtype not in _DTYPES:
            _fail("i8 moe to %s", dtype)
        q = xs.q
        _same_device(self.banks[0].q, q, logits)
        if _elsewhere(q):
            with torch.cuda.device(q.device):
                return self.forward(xs, logits, dtype)
        d = ctypes.byref(self.desc)
        need = lib().cw_i8_moe_workspace_size(d, t)
        if need == 0 and t > 0:
            raise CwError(CW_EINVAL, lib().cw_last_error().decode(errors="replace"))
        out = q.new_empty((t, self.hidden), dtype=dtype)
        ids = q.new_empty((t, self.top_k), dtype=torch.int32)
        w = q.new_empty((t, self.top_k), dtype=torch.float32)
        ws = q.new_empty(need)
        check(lib().cw_i8_moe_layer(d, q.data_ptr(), xs.scale.data_ptr(), logits.data_ptr(), t, _DTYPES[dtype], out.data_ptr(), ids.data_ptr(),
                                    w.data_ptr(), ws.data_ptr(), need, _stream(q)))
        return out, ids, w
