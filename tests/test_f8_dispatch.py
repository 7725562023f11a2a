"""Every kernel that the 8-bit float products can take is taken by some sizes, and by the sizes that the GPU tests run (CPU only)."""
import pytest

from tests.f8_rules import CUS, product, rules

EVERY = {False: {("few", g) for g in range(1, 5)} | {("tile", t) for t in (64, 128, 256)}, True: {("few", g) for g in range(1, 6)} | {("tile", t) for t in (64, 128, 256)}}
# sizes of every kernel, which tests/test_gpu_f8_instances.py runs: (exact, m, n, k)
INSTANCES = [(False, 16, 300, 260), (False, 31, 5000, 130), (False, 47, 4000, 300), (False, 63, 2000, 1000), (False, 120, 700, 400), (False, 500, 4100, 700), (False, 4090, 4091, 2000),
             (True, 16, 300, 260), (True, 31, 5000, 130), (True, 47, 4000, 300), (True, 63, 2000, 1000), (True, 79, 2500, 500), (True, 120, 700, 400), (True, 500, 4100, 700),
             (True, 4090, 4091, 1000)]


@pytest.mark.parametrize("exact", [False, True])
def test_every_kernel_is_reached(exact):
    assert {product(*i) for i in INSTANCES if i[0] == exact} == EVERY[exact]


@pytest.mark.parametrize("exact", [False, True])
def test_sizes_stay_among_them(exact):
    seen = {product(exact, m, n, k) for m in (1, 15, 17, 33, 49, 65, 81, 129, 300, 1000, 3000, 20000) for n in (1, 100, 2048, 2049, 4096, 4097, 30000) for k in (1, 300, 4096, 32768)}
    assert seen <= EVERY[exact]


def test_results_too_large_for_a_launch():
    assert product(False, 1 << 30, 1 << 26, 128) is None and product(False, 1 << 16, 1 << 20, 128) is not None


def test_groups_of_the_experts():
    r = rules()
    assert r.four_groups(128, 8192, 2880, CUS) and r.four_groups(256, 8192, 512, CUS)
    assert not r.four_groups(8, 4096, 4096, CUS)  # 512 picks an expert
    assert not r.four_groups(256, 4096, 1024, CUS)  # 16
    assert not r.four_groups(64, 4096, 1024, CUS)  # 256 blocks


# (exact, tokens, experts, picks a token, n, k) of every kernel of the experts' products, which tests/test_gpu_f8_instances.py runs
EXPERTS = {"two": [(False, 37, 8, 2, 300, 260), (True, 200, 8, 4, 300, 260)], "four": [(False, 2100, 256, 4, 300, 260), (True, 2100, 256, 4, 300, 260)],
           "tiles": [(False, 131, 4, 2, 300, 260), (True, 131, 2, 2, 300, 260), (False, 1000, 5, 3, 129, 1000), (True, 1000, 5, 3, 129, 1000)]}


def experts_form(exact, t, e, kp, n, k):
    r = rules()
    return "tiles" if r.sorted_tiles(exact, e, t * kp, n, CUS) else "four" if r.four_groups_of(e, t * kp, n, k, CUS) else "two"


@pytest.mark.parametrize("form", EXPERTS)
def test_every_kernel_of_the_experts_is_reached(form):
    assert {experts_form(*i) for i in EXPERTS[form]} == {form}


@pytest.mark.parametrize("exact", [0, 1])
def test_few_experts_of_many_picks_take_tiles(exact):
    r = rules()
    few = 127 if exact else 63  # picks an expert, one under the least
    assert r.sorted_tiles(exact, 8, 4096, 4096, CUS) and r.sorted_tiles(exact, 8, 8 * (few + 1), 4096, CUS) and not r.sorted_tiles(exact, 8, 8 * few, 4096, CUS)
    assert r.sorted_tiles(exact, 64, 64 * 200, 12 * 128, CUS) and not r.sorted_tiles(exact, 64, 64 * 200, 12 * 128 + 1, CUS)  # three blocks of W to a CU


def test_four_groups_end_sooner_with_a_long_k():
    r = rules()
    assert r.four_groups_of(128, 8192, 2880, 2880, CUS) and not r.four_groups_of(128, 8193, 2880, 2880, CUS)
    assert r.four_groups_of(128, 16384, 2880, 2048, CUS) and not r.four_groups_of(128, 16385, 2880, 2048, CUS)
