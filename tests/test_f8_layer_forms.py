"""Which of their two forms layers of 8-bit float experts take, and that the GPU tests' sizes take every kernel of both (CPU only)."""
import itertools

import pytest

from tests.f8_layer_rules import FEW, GROUPED, down_form, few, few_kernels

# (tokens, experts, top-k, hidden, inter), measured: two launches / grouped, us
MEASURED = [((8, 256, 8, 2048, 512), 42, 57), ((20, 256, 8, 2048, 512), 85, 93), ((48, 256, 8, 2048, 512), 182, 152), ((4, 128, 4, 2880, 2880), 88, 104), ((8, 128, 4, 2880, 2880), 161, 152),
            ((4, 8, 2, 2048, 4096), 40, 53), ((8, 8, 2, 2048, 4096), 68, 58), ((6, 64, 6, 2048, 1408), 70, 76), ((8, 64, 6, 2048, 1408), 89, 83), ((4, 16, 2, 4096, 2880), 66, 71), ((6, 16, 2, 4096, 2880), 95, 89),
            ((24, 64, 8, 1024, 256), 33, 36), ((32, 64, 8, 1024, 256), 41, 36), ((48, 16, 4, 256, 200), 22, 24), ((96, 16, 4, 256, 200), 37, 25), ((256, 16, 4, 256, 200), 87, 28), ((64, 64, 1, 512, 512), 24, 27),
            ((256, 64, 1, 512, 512), 75, 29), ((64, 1024, 2, 256, 128), 15, 26), ((512, 1024, 2, 256, 128), 85, 54)]


@pytest.mark.parametrize("size,two,grouped", [m for m in MEASURED if max(m[1:]) > 1.1 * min(m[1:])])
def test_the_faster_form_is_taken(size, two, grouped):
    assert few(*size) == (two < grouped)


def test_one_token_takes_two_launches_where_they_hold_it():
    for e, kp, h, i in itertools.product((1, 8, 64, 256, 1024), (1, 2, 8, 32), (16, 300, 4096), (1, 100, 512, 2880, 14336)):
        if kp <= e:
            assert few(1, e, kp, h, i) == (kp * ((i + 127) // 128 * 128) <= 16384)
    assert not few(1, 8, 2, 4097, 512)


def test_the_tests_sizes_take_every_kernel():
    assert all(few(*s) for s in FEW)
    took = [set(x) for x in zip(*(few_kernels(*s) for s in FEW))]
    assert took == [{4, 8, 16}, {2, 4, 6, 8}, {1, 2, 4, 8, 12, 16}]
    for form, sizes in GROUPED.items():
        for s in sizes:
            assert not few(*s)
            assert {down_form(exact, *s) for exact in (0, 1)} == {form}
