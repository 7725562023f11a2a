"""Which sizes the 8-bit product takes and which it refuses, on the host: a call with null pointers is refused for its size
(CW_ENOTSUP) or, where a kernel takes the size, for its pointers (CW_EINVAL). And that the sizes of the GPU tests take every
kernel instance, by the rules themselves."""
import pytest

import coachwhip_amd as cw
from coachwhip_amd import formats as F
from coachwhip_amd._lib import CW_EINVAL, CW_ENOTSUP

from . import i8_rules as rules
from .test_gpu_i8 import MM_SHAPES
from .test_gpu_i8_batch import BATCHES, K, N
from .test_gpu_i8_instances import DOWN, GATEUP, GROUPED, all_counts
from .test_gpu_i8_scales import SHAPES as SCALE_SHAPES


def size_status(m, n, k):
    return cw.lib().cw_i8_matmul(None, None, n, k, None, None, m, None, F.F32, None, n, None)


# a launch holds fewer than 2^22 tiles: of 256 x 256 where smaller tiles, though estimated faster, would be too many
@pytest.mark.parametrize("m,n,k,status", [
    ((1 << 28) + 1, 64, 512, CW_EINVAL), ((1 << 28) + 1, 64, 128, CW_EINVAL), ((1 << 29) + 1, 64, 512, CW_EINVAL), ((1 << 30) - 256, 64, 64, CW_EINVAL),
    ((1 << 30) - 256, 256, 64, CW_EINVAL), (1 << 30, 256, 64, CW_ENOTSUP), (1 << 30, 1, 1, CW_ENOTSUP), (1 << 24, 1 << 15, 128, CW_ENOTSUP),
    (1 << 21, 1 << 17, 64, CW_ENOTSUP), ((1 << 21) - 256, 1 << 17, 64, CW_EINVAL), (70, 1 << 26, 32768, CW_EINVAL), (70, (1 << 26) + 1, 64, CW_ENOTSUP),
    (1 << 12, 1 << 26, 64, CW_ENOTSUP), (1, 1 << 26, 64, CW_EINVAL)])
def test_products_of_many_tiles(m, n, k, status):
    assert size_status(m, n, k) == status


def test_every_product_kernel_is_tested():
    taken = {rules.product(*s) for s in MM_SHAPES}
    assert taken >= {("few", g) for g in (1, 2, 4)} | {("tile", *t) for t in ((64, 64), (64, 128), (128, 128), (256, 256))}
    taken = {rules.product(*s) for s in SCALE_SHAPES}
    assert taken >= {("few", g) for g in (1, 2, 4)} | {("tile", *t) for t in ((64, 64), (64, 128), (128, 128), (256, 256))}


def test_every_kernel_of_a_few_tokens_is_tested():
    taken = set().union(*[rules.layer(*c) for c in GATEUP + DOWN])
    want = {("gateup", w, n, r) for w in (4, 8, 16) for n in (1, 2, 3, 4) for r in (1, 2, 4) if not (r == 4 and n > 2)}
    want |= {("down", n, r) for n in (1, 2, 4, 8, 12, 16) for r in (1, 2, 4) if not (r == 4 and n > 4 or r == 2 and n > 8)}
    assert taken == want, (want - taken, taken - want)


def test_every_kernel_of_many_tokens_is_tested():
    """Both products, in tiles of every number of 16-pick groups, and every plan; more than one block of columns and step of k."""
    assert set().union(*[rules.layer(*c[:5]) for c in GROUPED]) == {("plan", w) for w in (0, 4, 8, 16)} | {("stream", g) for g in (2, 4)}
    for groups in (2, 4):
        cases = [c for c in GROUPED if ("stream", groups) in rules.layer(*c[:5])]
        assert {rules.row_groups(m) for c in cases for m in rules.tiles(all_counts(c[0], c[1], c[4], c[5]))} == {1, 2, 3, 4, 5, 6, 8}
        assert any(c[6] == "clamped" and c[7] for c in cases) and any(c[6] == "silu" for c in cases)
        assert any(c[3] > 64 * groups and c[2] > 128 * groups and c[2] % (64 * groups) and c[3] % (32 * groups) for c in cases)
    for E, K, _, _, T, counts, *_ in GROUPED:  # (picks that can be dealt out, each expert once a token)
        dealt = all_counts(E, K, T, counts)
        assert len(dealt) == E and sum(dealt) == T * K and min(dealt) >= 0 and max(dealt) <= T
    picks = [c[1] * c[4] for c in GROUPED if c[4] > 32]
    assert any(p <= 8192 for p in picks) and any(8192 < p <= 12288 for p in picks) and any(p > 12288 for p in picks)


@pytest.mark.parametrize("m,n,k,want", [
    ((1 << 28) + 1, 64, 512, ("tile", 128, 128)), ((1 << 30) - 256, 64, 64, ("tile", 256, 256)), (1 << 30, 256, 64, None)])
def test_tiles_beyond_a_launch_are_no_candidates(m, n, k, want):
    assert rules.product(m, n, k) == want


def test_batches_of_rows_take_every_product_kernel():
    assert {rules.product(m, N, K) for m in BATCHES + [5000]} | {rules.product(50, 300, K)} >= {("few", g) for g in (1, 2, 4)} | {
        ("tile", *t) for t in ((64, 64), (64, 128), (128, 128), (256, 256))}
