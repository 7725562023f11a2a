"""Which sizes the 8-bit product takes and which it refuses, on the host: a call with null pointers is refused for its size
(CW_ENOTSUP) or, where a kernel takes the size, for its pointers (CW_EINVAL)."""
import pytest

import coachwhip_amd as cw
from coachwhip_amd import formats as F
from coachwhip_amd._lib import CW_EINVAL, CW_ENOTSUP


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
