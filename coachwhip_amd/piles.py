"""Tokens sorted by expert and back, with weights applied, and the gradients of both.

- ``sort_picks``: the picks of a batch of tokens (``ops.route``'s ids) as piles, one per expert;
- ``to_piles`` / ``from_piles``: the tokens' rows to the piles, and the piles' rows back as each token's weighted sum
  (``ops.weighted_sum`` for rows that lie by expert);
- ``to_piles_grad`` / ``from_piles_grad``: their gradients, as functions of their own: nothing here records a graph of torch's.

No counterpart in the reference, whose piles exist inside its kernels only. Rows are f32, f16 or bf16 tensors, on the current
stream of their own device; all arithmetic runs in libcwmoe.so, in a fixed order: the same inputs give the same bits. Shape and
type errors raise ``CwError``.
"""
import functools
import operator
from dataclasses import dataclass
from typing import Optional

import torch

from . import ops
from ._lib import CW_EINVAL, CwError, check, lib
from .i8 import _DTYPES, _elsewhere, _fail, _floats, _ptr, _same_device, _stream


def _count(n, what):
    """n as an int that the library's calls take as it is."""
    try:
        i = operator.index(n)
    except TypeError:
        i = 0
    if not 0 < i < 1 << 31:
        _fail("%s: %r", what, n)
    return i


@dataclass
class Piles:
    """T tokens' K picks each, sorted by expert (``sort_picks`` makes them).

    ``order`` (T K,) int32: the pick (token * K + choice) at each position, an expert's in the order of the tokens; ``place``
    (T K,) int32: the position of each pick; ``offsets`` (n_experts + 1,) int32: the first position of each expert.
    Positions from ``offsets[n_experts]`` on are those of picks of no expert. ``tiles``: the products' plan."""
    order: torch.Tensor
    place: torch.Tensor
    offsets: torch.Tensor
    tiles: torch.Tensor
    tokens: int
    top_k: int
    n_experts: int


def sort_picks(ids: torch.Tensor, n_experts: int) -> Piles:
    """ids (T, K) int32, the experts of each token's picks: 0 .. n_experts - 1, or any other number (-1, say) for experts that
    another device holds."""
    n_experts = _count(n_experts, "experts")
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.dtype != torch.int32 or ids.dim() != 2 or not ids.is_contiguous():
        _fail("ids: a contiguous (tokens, picks) int32 device tensor")
    t, k = ids.shape
    if k == 0:
        _fail("ids of no picks")
    if _elsewhere(ids):
        with torch.cuda.device(ids.device):
            return sort_picks(ids, n_experts)
    n = t * k
    sizes, need = _sizes(n, n_experts)
    buf = ids.new_empty(sum(sizes))
    order, _, place, _, offsets, _, tiles, ws = buf.split_with_sizes(sizes)
    check(lib().cw_sort_picks(ids.data_ptr(), n, n_experts, order.data_ptr(), place.data_ptr(), offsets.data_ptr(), tiles.data_ptr(),
                              ws.data_ptr() if need else None, need, _stream(ids)))
    return Piles(order, place, offsets, tiles, t, k, n_experts)


@functools.lru_cache(maxsize=256)
def _sizes(picks, n_experts):
    """int32s of order, place, offsets, tiles (each in whole 16 bytes) and the workspace; the workspace's bytes."""
    size = lib().cw_pile_tiles_bytes(picks, n_experts)
    if size == 0:
        raise CwError(CW_EINVAL, lib().cw_last_error().decode(errors="replace"))
    need = lib().cw_sort_picks_workspace_size(picks, n_experts)
    return [picks, -picks % 4, picks, -picks % 4, n_experts + 1, -(n_experts + 1) % 4, size // 4, need // 4], need


def _rows(x, n, h, what):
    ld = _floats(x, what)
    if x.shape[0] != n or (h is not None and x.shape[1] != h):
        _fail("%s %s: expected %d rows%s", what, tuple(x.shape), n, "" if h is None else " of %d" % h)
    return ld


def to_piles(x: torch.Tensor, piles: Piles) -> torch.Tensor:
    """(T K, h): the row x[token] at each position, zeros at those of no expert. x (T, h), any stride between rows."""
    p = piles
    ld = _rows(x, p.tokens, None, "x")
    _same_device(x, p.place)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return to_piles(x, piles)
    h = x.shape[1]
    rows = x.new_empty((p.tokens * p.top_k, h))
    check(lib().cw_to_piles(_DTYPES[x.dtype], x.data_ptr(), ld, p.tokens, p.top_k, p.n_experts, h, p.order.data_ptr(), p.offsets.data_ptr(),
                            rows.data_ptr(), _stream(x)))
    return rows


def _weights(w, p):
    if w is not None:
        ops._need(w, torch.float32, "weights")
        if w.shape != (p.tokens, p.top_k):
            _fail("weights %s: expected (%d, %d)", tuple(w.shape), p.tokens, p.top_k)


def from_piles(rows: torch.Tensor, w: Optional[torch.Tensor], piles: Piles) -> torch.Tensor:
    """(T, h): sum over j of w[t][j] * rows[place of the pick], in f32 in the picks' order, rounded once to rows' type; w
    (T, K) f32, or None for ones. Picks of no expert add nothing, whatever their rows hold."""
    p = piles
    ld = _rows(rows, p.tokens * p.top_k, None, "rows")
    _weights(w, p)
    _same_device(rows, w, p.place)
    if _elsewhere(rows):
        with torch.cuda.device(rows.device):
            return from_piles(rows, w, piles)
    h = rows.shape[1]
    out = rows.new_empty((p.tokens, h))
    check(lib().cw_from_piles(_DTYPES[rows.dtype], rows.data_ptr(), ld, _ptr(w), p.tokens, p.top_k, p.n_experts, h, p.place.data_ptr(),
                              p.offsets.data_ptr(), out.data_ptr(), _stream(rows)))
    return out


def to_piles_grad(drows: torch.Tensor, piles: Piles) -> torch.Tensor:
    """The gradient of ``to_piles``' x, (T, h), from that of its rows."""
    return from_piles(drows, None, piles)


def from_piles_grad(dout: torch.Tensor, rows: torch.Tensor, w: torch.Tensor, piles: Piles):
    """(the gradient of ``from_piles``' rows, that of w (T, K) f32), from that of its output: w[t][j] * dout[t] at each pick's
    position and <dout[t], rows[position]>, zeros for picks of no expert."""
    p = piles
    ldd = _rows(dout, p.tokens, None, "dout")
    h = dout.shape[1]
    ldr = _rows(rows, p.tokens * p.top_k, h, "rows")
    if rows.dtype != dout.dtype:
        _fail("rows %s for dout %s", rows.dtype, dout.dtype)
    if w is None:
        _fail("from_piles_grad: weights of (%d, %d)", p.tokens, p.top_k)
    _weights(w, p)
    _same_device(dout, rows, w, p.place)
    if _elsewhere(dout):
        with torch.cuda.device(dout.device):
            return from_piles_grad(dout, rows, w, piles)
    drows = dout.new_empty((p.tokens * p.top_k, h))
    dw = w.new_empty((p.tokens, p.top_k))
    check(lib().cw_from_piles_grad(_DTYPES[dout.dtype], dout.data_ptr(), ldd, rows.data_ptr(), ldr, w.data_ptr(), p.tokens, p.top_k, p.n_experts, h,
                                   p.place.data_ptr(), p.offsets.data_ptr(), drows.data_ptr(), dw.data_ptr(), _stream(dout)))
    return drows, dw
