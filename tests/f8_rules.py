"""The rules by which the 8-bit float path picks its kernels (csrc/cw_f8_rules.h, plain C++), compiled for the host."""
import ctypes
import functools
import os
import subprocess
import tempfile

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "coachwhip_amd", "csrc")
SHIM = """
#include "cw_f8_rules.h"
extern "C" {
int few_groups(int exact, long m, long n, int cus) { return cw::f8_few_groups(exact, m, n, cus); }
int pick_tile(int exact, long m, long n, int rb, int cus) { return cw::f8_pick_tile(exact, m, n, rb, cus); }
int tile_rows(int i) { return cw::F8_TILES[0][i].tm; }
int four_groups(int E, long picks, long n, int cus) { return cw::f8_four_groups(E, picks, n, 2048, cus); }
int four_groups_of(int E, long picks, long n, long k, int cus) { return cw::f8_four_groups(E, picks, n, k, cus); }
int sorted_tiles(int exact, int E, long picks, long n, int cus) { return cw::f8_sorted_tiles(exact, E, picks, n, cus); }
}
"""
CUS = 256


@functools.lru_cache(None)
def rules():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "rules.cpp"), os.path.join(d, "rules.so")
        with open(src, "w") as f:
            f.write(SHIM)
        subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", out, src], check=True)
        lib = ctypes.CDLL(out)
    lib.few_groups.argtypes = [ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_int]
    lib.pick_tile.argtypes = [ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_int, ctypes.c_int]
    lib.four_groups.argtypes = [ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_int]
    lib.four_groups_of.argtypes = [ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_long, ctypes.c_int]
    lib.sorted_tiles.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_int]
    return lib


def product(exact, m, n, k):
    """The kernel of a product: ("few", groups of 16 rows), ("tile", its size), or None where no tile's count fits a launch."""
    r, rb = rules(), (k + 127) // 128 * 128
    few = r.few_groups(exact, m, n, CUS)
    if few:
        return "few", few
    tile = r.pick_tile(exact, m, n, rb, CUS)
    return ("tile", r.tile_rows(tile)) if tile >= 0 else None
