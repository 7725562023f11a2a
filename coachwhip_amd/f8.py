"""Experts in 8-bit floats: e4m3 codes with a scale for each block of 128, the format that checkpoints of large MoE models are
published in. Weights have a scale for each 128 x 128, activations one for each 128 columns of a row.

- ``quantize_f8`` / ``swiglu_f8``: rows of floats, or of a SwiGLU, as codes;
- ``F8MatMul``: codes times an ``F8Matrix``, beside ``ops.QMatMul`` and ``i8.I8MatMul``;
- ``F8ExpertMatMul``: the product of sorted rows (``piles.sort_picks``), each with its expert's matrix;
- ``F8MoeLayer``: a layer of such experts, beside ``ops.MoeLayer`` and ``i8.I8MoeLayer``.

A checkpoint's codes and scales are taken as they are (``F8Matrix``, ``F8ExpertBank``); ``from_qtensor`` and ``from_bank`` lay GGUF
weights out once, when a model is loaded. No counterpart in the reference. Activations are f32, f16 or bf16 tensors, on the
current stream of their own device; all arithmetic runs in libcwmoe.so. Shape and type errors raise ``CwError``.
"""
import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import formats as F
from . import ops
from ._lib import CW_EINVAL, CW_F8_MAX_K, CwError, F8MoeDesc, check, lib
from .i8 import _DTYPES, _SILU, _elsewhere, _fail, _floats, _ptr, _same_device, _stream, _vector, row_bytes
from .piles import Piles, _count

_E4M3 = torch.float8_e4m3fn


def blocks(n: int) -> int:
    """Blocks of 128 that n rows or columns take."""
    return (n + 127) // 128


def _codes(q, scale, k, lead, what):
    k = _count(k, "codes of a row")
    if not isinstance(q, torch.Tensor) or not isinstance(scale, torch.Tensor) or not q.is_cuda or q.dtype != _E4M3 or scale.dtype != torch.float32:
        _fail("%s: float8_e4m3fn codes and f32 scales on a device", what)
    if q.device != scale.device or not q.is_contiguous() or not scale.is_contiguous():
        _fail("%s: contiguous codes and scales on one device", what)
    shape = q.shape
    if len(shape) != lead + 1 or shape[-1] != row_bytes(k):
        _fail("%s codes %s: rows of %d bytes for %d codes", what, tuple(shape), row_bytes(k), k)
    if q.data_ptr() % 16:
        _fail("%s codes must be 16-byte aligned", what)


def _matrix(q, scale, k, lead, what):
    _codes(q, scale, k, lead, what)
    want = (*q.shape[:-2], blocks(q.shape[-2]), blocks(k))
    if scale.shape != want:
        _fail("%s scales %s for codes %s: expected %s", what, tuple(scale.shape), tuple(q.shape), want)


@dataclass
class F8Rows:
    """Rows of k codes: ``q`` (rows, row_bytes(k)) e4m3, zeros past k, and ``scale`` (blocks(k), rows) f32."""
    q: torch.Tensor
    scale: torch.Tensor
    k: int

    def __post_init__(self):
        _codes(self.q, self.scale, self.k, 1, "rows")
        if self.scale.shape != (blocks(self.k), self.q.shape[0]):
            _fail("rows scales %s for codes %s: expected (%d, %d)", tuple(self.scale.shape), tuple(self.q.shape), blocks(self.k), self.q.shape[0])

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
        check(lib().cw_dequantize_f8(q.data_ptr(), self.scale.data_ptr(), rows, self.k, _DTYPES[dtype], out.data_ptr(), _stream(q)))
        return out


def _new_rows(x, rows, k):
    if k > CW_F8_MAX_K:
        _fail("rows of %d codes above %d", k, CW_F8_MAX_K)
    r = object.__new__(F8Rows)
    r.q, r.scale, r.k = x.new_empty((rows, row_bytes(k)), dtype=_E4M3), x.new_empty((blocks(k), rows), dtype=torch.float32), k
    return r


def quantize_f8(x: torch.Tensor) -> F8Rows:
    """Rows (any stride between them) as codes: of each 128 columns scale = max|x| / 448, code = x / scale to the nearest."""
    ld = _floats(x, "x")
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return quantize_f8(x)
    rows, k = x.shape
    r = _new_rows(x, rows, k)
    check(lib().cw_quantize_f8(_DTYPES[x.dtype], x.data_ptr(), ld, rows, k, r.q.data_ptr(), r.scale.data_ptr(), _stream(x)))
    return r


def swiglu_f8(g: torch.Tensor, u: torch.Tensor, act: Optional[ops.ExpertAct] = None) -> F8Rows:
    """silu(g) * u, or the clamped SwiGLU of ``act``, as codes. g and u: rows of one type and stride (the
    halves of one product's rows). Biases belong to the product (``F8MatMul``): ``act`` must have none."""
    act = act or _SILU
    if act.gate_b is not None or act.up_b is not None or act.down_b is not None or act.pad:
        _fail("swiglu_f8: an activation with biases or padding")
    ld = _floats(g, "gate")
    if _floats(u, "up") != ld or u.dtype != g.dtype or u.shape != g.shape:
        _fail("gate %s %s and up %s %s differ in shape, type or stride", tuple(g.shape), g.dtype, tuple(u.shape), u.dtype)
    _same_device(g, u)
    if _elsewhere(g):
        with torch.cuda.device(g.device):
            return swiglu_f8(g, u, act)
    rows, k = g.shape
    r = _new_rows(g, rows, k)
    check(lib().cw_swiglu_f8(_DTYPES[g.dtype], g.data_ptr(), u.data_ptr(), ld, rows, k, act.kind, act.alpha, act.limit, r.q.data_ptr(),
                             r.scale.data_ptr(), _stream(g)))
    return r


def _quantize_matrix(w, q, scale):
    ld = _floats(w, "weights")
    n, k = w.shape
    if k > CW_F8_MAX_K:
        _fail("rows of %d codes above %d", k, CW_F8_MAX_K)
    with torch.cuda.device(w.device):
        check(lib().cw_quantize_f8_matrix(_DTYPES[w.dtype], w.data_ptr(), ld, n, k, q.data_ptr(), scale.data_ptr(), _stream(w)))


@dataclass
class F8Matrix:
    """An (n, k) weight: ``q`` (n, row_bytes(k)) e4m3, zeros past k, and ``scale`` (blocks(n), blocks(k)) f32."""
    q: torch.Tensor
    scale: torch.Tensor
    k: int

    def __post_init__(self):
        _matrix(self.q, self.scale, self.k, 1, "matrix")

    @property
    def shape(self):
        return self.q.shape[0], self.k

    @classmethod
    def from_float(cls, w: torch.Tensor):
        """Of (n, k) floats, each 128 x 128 as ``quantize_f8`` has 128 columns of a row."""
        _floats(w, "weights")
        n, k = w.shape
        q, scale = w.new_empty((n, row_bytes(k)), dtype=_E4M3), w.new_empty((blocks(n), blocks(k)), dtype=torch.float32)
        _quantize_matrix(w, q, scale)
        return cls(q, scale, k)

    @classmethod
    def from_qtensor(cls, w: ops.QTensor):
        with torch.cuda.device(w.data.device):
            return cls.from_float(w.dequantize())


class F8MatMul:
    """y = x . W^T (+ bias) for rows of codes x and a matrix of codes W, in f32, rounded once to the type asked for. Products are exact for f32
    and f16; for bf16 the 8-bit matrix instruction's, 1.5e-5 of a result of random codes (7 * 2^-13 of the terms' magnitudes at most)."""

    def __init__(self, matrix: F8Matrix, bias: Optional[torch.Tensor] = None):
        _vector(bias, matrix.shape[0], "bias")
        _same_device(matrix.q, bias)
        self.w, self.bias = matrix, bias

    def forward(self, xs: F8Rows, dtype=torch.float32) -> torch.Tensor:
        w, q, k = self.w.q, xs.q, xs.k
        if k != self.w.k:
            _fail("rows of %d incompatible with %s", k, self.w.shape)
        if dtype not in _DTYPES:
            _fail("f8 matmul to %s", dtype)
        _same_device(w, q)
        if _elsewhere(q):
            with torch.cuda.device(q.device):
                return self.forward(xs, dtype)
        m, n = q.shape[0], w.shape[0]
        y = q.new_empty((m, n), dtype=dtype)
        check(lib().cw_f8_matmul(w.data_ptr(), self.w.scale.data_ptr(), n, k, q.data_ptr(), xs.scale.data_ptr(), m, _ptr(self.bias),
                                 _DTYPES[dtype], y.data_ptr(), n, _stream(q)))
        return y

    __call__ = forward


@dataclass
class F8ExpertBank:
    """One matrix of every expert: ``q`` (experts, n, row_bytes(k)) e4m3, ``scale`` (experts, blocks(n), blocks(k)) f32."""
    q: torch.Tensor
    scale: torch.Tensor
    k: int

    def __post_init__(self):
        _matrix(self.q, self.scale, self.k, 2, "bank")

    @property
    def n(self):
        return self.q.shape[1]

    @classmethod
    def _new(cls, e, n, k, device):
        return (torch.empty((e, n, row_bytes(k)), dtype=_E4M3, device=device), torch.empty((e, blocks(n), blocks(k)), dtype=torch.float32, device=device))

    @classmethod
    def from_float(cls, w: torch.Tensor):
        """Of (experts, n, k) floats."""
        if not isinstance(w, torch.Tensor) or w.dim() != 3:
            _fail("bank: (experts, n, k) weights, got %s", tuple(w.shape) if isinstance(w, torch.Tensor) else type(w))
        q, scale = cls._new(*w.shape, w.device)
        for e in range(w.shape[0]):
            _quantize_matrix(w[e], q[e], scale[e])
        return cls(q, scale, w.shape[2])

    @classmethod
    def from_bank(cls, bank: ops.ExpertBank):
        """Of a bank of GGUF blocks, one expert's floats at a time."""
        n, k = bank.n, bank.k
        q, scale = cls._new(bank.n_slots, n, k, bank.data.device)
        size = F.matrix_bytes(bank.dtype, n, k)
        with torch.cuda.device(bank.data.device):
            for s in range(bank.n_slots):
                raw = bank.data[s * bank.slot_stride:s * bank.slot_stride + size]
                _quantize_matrix(ops.dequantize(bank.dtype, raw, n * k).view(n, k), q[s], scale[s])
        return cls(q, scale, k)


class F8ExpertMatMul:
    """y[pos] = x_row . W[expert of pos]^T (+ bias[expert]) for the positions of ``piles.sort_picks``, zeros at those of no expert."""

    def __init__(self, bank: F8ExpertBank, bias: Optional[torch.Tensor] = None):
        _vector(bias, bank.q.shape[0] * bank.n, "bias")
        _same_device(bank.q, bias)
        self.bank, self.bias = bank, bias

    def forward(self, xs: F8Rows, piles: Piles, dtype=torch.float32, by_token: bool = False) -> torch.Tensor:
        """xs: a row for each position, or with ``by_token`` one for each token (a position's is its token's). (T K, n)."""
        b, q, p = self.bank, xs.q, piles
        picks, m, n = p.tokens * p.top_k, q.shape[0], b.n
        if xs.k != b.k or m != (p.tokens if by_token else picks):
            _fail("%d rows of %d for %d tokens of %d picks and experts (%d, %d)", m, xs.k, p.tokens, p.top_k, n, b.k)
        if p.n_experts != b.q.shape[0]:
            _fail("piles of %d experts for a bank of %d", p.n_experts, b.q.shape[0])
        if dtype not in _DTYPES:
            _fail("f8 matmul to %s", dtype)
        _same_device(b.q, q, p.place)
        if _elsewhere(q):
            with torch.cuda.device(q.device):
                return self.forward(xs, piles, dtype, by_token)
        y = q.new_empty((picks, n), dtype=dtype)
        check(lib().cw_f8_matmul_experts(b.q.data_ptr(), b.q.stride(0), b.scale.data_ptr(), p.n_experts, n, b.k, q.data_ptr(), xs.scale.data_ptr(), m,
                                         p.order.data_ptr() if by_token else None, p.top_k, picks, p.tiles.data_ptr(), _ptr(self.bias),
                                         _DTYPES[dtype], y.data_ptr(), n, _stream(q)))
        return y

    __call__ = forward


class F8MoeLayer:
    """A MoE layer of experts in 8-bit floats, all resident: ``ops.MoeLayer`` on rows of codes. Products as ``F8MatMul`` has them for the type asked for."""

    def __init__(self, gate: F8ExpertBank, up: F8ExpertBank, down: F8ExpertBank, top_k: int, norm_topk_prob: bool = True,
                 act: Optional[ops.ExpertAct] = None):
        act, top_k = act or _SILU, _count(top_k, "top_k")
        e, inter, hidden = gate.q.shape[0], gate.n, gate.k
        for b, n, k, what in ((up, inter, hidden, "up"), (down, hidden, inter, "down")):
            if b.q.shape[0] != e or b.n != n or b.k != k:
                _fail("%s bank of %d (%d, %d) for %d experts (%d, %d)", what, b.q.shape[0], b.n, b.k, e, n, k)
        if act.pad not in (0, inter):
            _fail("f8 moe: padding (rows of codes are padded by themselves)")
        biases = (act.gate_b, act.up_b, act.down_b)
        for b, n, what in zip(biases, (inter, inter, hidden), ("gate", "up", "down")):
            _vector(b, e * n, "%s bias" % what)
        _same_device(gate.q, up.q, down.q, *biases)
        self.banks, self.act = (gate, up, down), act
        self.n_experts, self.top_k, self.hidden, self.inter = e, top_k, hidden, inter
        d = F8MoeDesc()
        d.n_experts, d.top_k, d.hidden, d.inter, d.norm = e, top_k, hidden, inter, int(norm_topk_prob)
        d.act, d.alpha, d.limit = act.kind, act.alpha, act.limit
        for m, b in enumerate(self.banks):
            d.w[m], d.scale[m], d.slot_stride[m] = b.q.data_ptr(), b.scale.data_ptr(), b.q.stride(0)
            d.bias[m] = None if biases[m] is None else biases[m].data_ptr()
        self.desc = d

    def forward(self, xs: F8Rows, logits: torch.Tensor, dtype=torch.float32):
        """xs T rows of hidden, logits (T, E) f32 -> (out (T, hidden), ids (T, K), w (T, K)). The workspace is
        allocated for the call (on the stream, or in the graph that captures it)."""
        ops._need(logits, torch.float32, "logits")
        t = len(xs)
        if xs.k != self.hidden or logits.shape != (t, self.n_experts):
            _fail("rows of %d / logits %s do not fit the layer", xs.k, tuple(logits.shape))
        if dtype not in _DTYPES:
            _fail("f8 moe to %s", dtype)
        q = xs.q
        _same_device(self.banks[0].q, q, logits)
        if _elsewhere(q):
            with torch.cuda.device(q.device):
                return self.forward(xs, logits, dtype)
        d = ctypes.byref(self.desc)
        need = lib().cw_f8_moe_workspace_size(d, t)
        if need == 0 and t > 0:
            raise CwError(CW_EINVAL, lib().cw_last_error().decode(errors="replace"))
        out = q.new_empty((t, self.hidden), dtype=dtype)
        ids = q.new_empty((t, self.top_k), dtype=torch.int32)
        w = q.new_empty((t, self.top_k), dtype=torch.float32)
        ws = q.new_empty(need, dtype=torch.uint8)
        check(lib().cw_f8_moe_layer(d, q.data_ptr(), xs.scale.data_ptr(), logits.data_ptr(), t, _DTYPES[dtype], out.data_ptr(), ids.data_ptr(),
                                    w.data_ptr(), ws.data_ptr(), need, _stream(q)))
        return out, ids, w
