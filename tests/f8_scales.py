"""Codes and scales whose product of two scales, or whose sums on the way, leave f32's range while the results do not, and the
results in 64 bits. On any device: inputs are made on the host from their seed."""
import torch

E4M3 = torch.float8_e4m3fn
U = 2.0 ** -24

# zeros: the last block of k has zero codes in x and scales whose product overflows: nothing, and no infinity times zero
# tiny: its codes are the smallest ones, so that the result is about 2^114
# under: every product of scales is below 2^-150, which f32 rounds to zero, and the sums are about 2^24
# cancel: two blocks' parts, each beyond f32, are one the other's negative: exactly, whatever the order, as their codes are small integers
KINDS = {"zeros": (torch.float32, torch.float16, torch.bfloat16), "tiny": (torch.float32, torch.bfloat16), "under": (torch.float32, torch.bfloat16),
         "cancel": (torch.float32, torch.float16, torch.bfloat16)}
USUAL = 47  # cancel: the largest power of two of a scale that takes no second way; with it the parts stay in f32


def blocks(n):
    return (n + 127) // 128


def strange_rows(m):
    return (torch.arange(m) % 3 == 1) | (torch.arange(m) == m - 1)


def strange_columns(n):
    """Of blocks of 128 columns: every second, and the last."""
    at = torch.arange(blocks(n))
    return (at % 2 == 1) | (at == blocks(n) - 1)


def operands(kind, m, n, k, seed, experts=1, power=62):
    """(codes of x, its scales, codes of the experts' matrices, their scales): the first of several experts has usual scales."""
    g = torch.Generator().manual_seed(seed)
    kb, nb = blocks(k), blocks(n)
    x, w = torch.zeros(m, 128 * kb), torch.zeros(experts, n, 128 * kb)
    x[:, :k], w[..., :k] = torch.randn(m, k, generator=g) * 100, torch.randn(experts, n, k, generator=g) * 100
    sx, sw = 0.004 + 0.003 * torch.rand(kb, m, generator=g), 0.004 + 0.003 * torch.rand(experts, nb, kb, generator=g)
    rows, cols, first = strange_rows(m), strange_columns(n), 1 if experts > 1 else 0
    last = 128 * (kb - 1)
    factor = {"zeros": 2.0 ** 74, "tiny": 2.0 ** 72, "under": 2.0 ** -69}.get(kind)
    if kind == "zeros":
        x[:, last:] = 0
    elif kind == "tiny":
        sign = lambda *s: (2 * torch.randint(0, 2, s, generator=g) - 1).float()
        x[:, last:k], w[..., last:k] = 2.0 ** -9 * sign(m, k - last), 2.0 ** -9 * sign(experts, n, k - last)
    elif kind == "under":
        x[:, :k], w[..., :k] = 300 + x[:, :k].abs(), 300 + w[..., :k].abs()
    else:
        same = min(128, k - 128)
        small = lambda *s: 2.0 ** torch.randint(2, 5, s, generator=g)
        x[:, :256], w[..., :256] = 0, 0
        x[:, :same], w[..., :same] = small(m, same), small(experts, n, same)
        x[:, 128:128 + same], w[..., 128:128 + same] = -x[:, :same], w[..., :same]
    if kind in ("zeros", "tiny"):
        sx[-1, rows] *= factor
        sw[first:, cols, -1] *= factor
    elif kind == "under":
        sx[:, rows] *= factor
        sw[first:, cols] *= factor
    else:
        sx[:2], sw[..., :2] = 2.0 ** power, 2.0 ** power
    return x.clamp(-448, 448).to(E4M3), sx, w.clamp(-448, 448).to(E4M3), sw


def result(kind, xq, sx, wq, sw, k, dtype, bias=None):
    """One matrix's product in 64 bits, and how far a result of the type may be: of each block's terms' magnitudes 2 U for each of 128
    products, a rounding for each block and 16 that join them, for bf16 also what the 8-bit instruction leaves out: it cuts 7 of 8
    neighbouring products to multiples of 2^-13 of the largest's power of two, 7 * 2^-13 of the sum at most; nothing for the parts of
    `cancel` that are exact; the rounding to the type."""
    n, kb = wq.shape[0], sw.shape[1]
    want = torch.zeros(xq.shape[0], n, dtype=torch.float64, device=xq.device)
    off = torch.zeros_like(want)
    rel = (2 * 128 + kb + 16) * U + (7 * 2.0 ** -13 if dtype == torch.bfloat16 else 0.0)
    for b in range(kb):
        at = slice(128 * b, 128 * (b + 1))
        xv, wv = xq[:, at].double(), wq[:, at].double()
        s = sx[b].double()[:, None] * sw[:, b].double().repeat_interleave(128)[:n]
        want += (xv @ wv.t()) * s
        if kind != "cancel" or b > 1:
            off += rel * (xv.abs() @ wv.abs().t()) * s
    if bias is not None:
        want = want + bias.double()
        off += U * (want.abs() + bias.double().abs())
    info = torch.finfo(dtype)
    return want, off + info.eps / 2 * (want.abs() + off) + info.smallest_normal * info.eps


def in_f32(xq, sx, wq, sw):
    """The formula with every product of scales and every sum in f32, as it would be without a second way for strange scales."""
    n = wq.shape[0]
    acc = torch.zeros(xq.shape[0], n)
    for b in range(sw.shape[1]):
        at = slice(128 * b, 128 * (b + 1))
        p = xq[:, at].float() @ wq[:, at].float().t()
        acc = acc + p * (sx[b][:, None] * sw[:, b].repeat_interleave(128)[:n])
    return acc
