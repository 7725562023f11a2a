"""The rules by which the 8-bit integer path picks its kernels (csrc/cw_i8_rules.h, plain C++), compiled for the host."""
import ctypes
import functools
import os
import subprocess
import tempfile

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "coachwhip_amd", "csrc")
SHIM = """
#include "cw_i8_rules.h"
extern "C" {
int few_groups(long m, long n, int rb) { return cw::i8_few_groups(m, n, rb); }
int pick_tile(long m, long n, int rb, int cus) { return cw::i8_pick_tile(m, n, rb, cus); }
int tile_rows(int i) { return cw::I8_TILES[i].tm; }
int tile_columns(int i) { return cw::I8_TILES[i].tn; }
int few_tokens(int E, int K, int H, int I, int T) { return cw::i8_few_tokens(E, K, H, I, T); }
int route_width(int E) { return cw::i8_route_width(E); }
int gateup_pieces(int rbh) { return cw::i8_gateup_pieces(rbh); }
int gateup_rows(int pieces, int I, long picks, int cus) { return cw::i8_gateup_rows(pieces, I, picks, cus); }
int down_pieces(int K, int rbi) { return cw::i8_down_pieces(K, rbi); }
int down_rows(int pieces, int H, long T, int cus) { return cw::i8_down_rows(pieces, H, T, cus); }
int many_picks(int E, int K, int I, int T, int cus) { return cw::i8_many_picks(E, K, I, T, cus); }
int plan_tokens() { return cw::I8_PLAN_TOKENS; }
int tile_picks() { return cw::I8_TILE; }
}
"""
CUS = 256


def row_bytes(k):
    return (k + 127) // 128 * 128


@functools.lru_cache(None)
def rules():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "rules.cpp"), os.path.join(d, "rules.so")
        with open(src, "w") as f:
            f.write(SHIM)
        subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", out, src], check=True)
        lib = ctypes.CDLL(out)
    for name in ("few_groups", "pick_tile"):
        getattr(lib, name).argtypes = [ctypes.c_long, ctypes.c_long] + [ctypes.c_int] * (1 + (name == "pick_tile"))
    lib.gateup_rows.argtypes = lib.down_rows.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_long, ctypes.c_int]
    return lib


def product(m, n, k):
    """The kernel of a product: ("few", groups of 16 rows) or ("tile", rows, columns)."""
    r, rb = rules(), row_bytes(k)
    few = r.few_groups(m, n, rb)
    if few:
        return "few", few
    tile = r.pick_tile(m, n, rb, CUS)
    return ("tile", r.tile_rows(tile), r.tile_columns(tile)) if tile >= 0 else None


def layer(E, K, H, I, T):
    """The kernels of a layer: gate and up's and down's of a few tokens, or the plan's and the grouped products'."""
    r = rules()
    if r.few_tokens(E, K, H, I, T):
        g, d = r.gateup_pieces(row_bytes(H)), r.down_pieces(K, row_bytes(I))
        return {("gateup", r.route_width(E), g, r.gateup_rows(g, I, T * K, CUS)), ("down", d, r.down_rows(d, H, T, CUS))}
    return {("plan", r.route_width(E) if T <= r.plan_tokens() else 0), ("stream", 4 if r.many_picks(E, K, I, T, CUS) else 2)}


def tiles(counts):
    """The sizes of the tiles of experts with these numbers of picks: spread evenly, in whole 16s."""
    out = []
    for c in counts:
        n = -(-c // rules().tile_picks())
        rows = (-(-c // n) + 15) // 16 * 16 if n else 0
        out += [min(rows, c - q * rows) for q in range(n)]
    return out


def row_groups(m):
    """Groups of 16 picks that the grouped products' loop of a tile of m picks holds."""
    return 8 if m > 96 else (m + 15) // 16
