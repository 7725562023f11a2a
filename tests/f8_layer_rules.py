"""The rule by which layers of 8-bit float experts pick their form (csrc/cw_f8_rules.h), compiled for the host, and the sizes of the
GPU tests of every kernel that a layer can take."""
import ctypes
import functools
import os
import subprocess
import tempfile

from tests.f8_rules import CSRC, CUS, rules

SHIM = """
#include "cw_f8_rules.h"
extern "C" int few_tokens(int E, int K, int H, int I, int T) { return cw::f8_few_tokens(E, K, H, I, T); }
"""


@functools.lru_cache(None)
def layer_rules():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "rules.cpp"), os.path.join(d, "rules.so")
        with open(src, "w") as f:
            f.write(SHIM)
        subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", out, src], check=True)
        return ctypes.CDLL(out)


def few(t, e, kp, h, i):
    return bool(layer_rules().few_tokens(e, kp, h, i, t))


def down_form(exact, t, e, kp, h, i):
    """The kernel of a grouped layer's down: its hidden rows are f32, of exact products or of the 8-bit instruction's."""
    r = rules()
    return "tiles" if r.sorted_tiles(exact, e, t * kp, h, CUS) else "four" if r.four_groups_of(e, t * kp, h, i, CUS) else "two"


def steps(n, of):
    """The number of steps that a kernel is built for, of `of`, that holds n."""
    return next(s for s in of if n <= s)


def few_kernels(t, e, kp, h, i):
    """(logits of a lane, steps of gate and up, steps of down) of the two launches."""
    width = 4 if e <= 256 else 8 if e <= 512 else 16
    up, down = (h + 127) // 128, kp * ((i + 127) // 128)
    return width, steps((up + 3) // 4, (2, 4, 6, 8)), steps((down + 7) // 8, (1, 2, 4, 8, 12, 16))


# (tokens, experts, top-k, hidden, inter)
FEW = [(1, 8, 1, 1000, 100), (3, 8, 2, 1100, 500), (2, 300, 4, 2100, 1000), (2, 600, 5, 4000, 1200), (2, 1024, 6, 300, 2000), (1, 40, 32, 500, 500), (1, 8, 7, 4096, 2300),
       (2, 40, 6, 4000, 700), (1, 600, 4, 2500, 300), (17, 16, 4, 256, 200)]
GROUPED = {"two": [(100, 8, 2, 300, 260), (64, 64, 6, 2048, 300), (3, 16, 2, 4200, 300)], "four": [(2100, 256, 4, 300, 260), (2048, 128, 4, 1100, 2200)],
           "tiles": [(700, 4, 2, 384, 1000), (700, 16, 4, 256, 200)]}
