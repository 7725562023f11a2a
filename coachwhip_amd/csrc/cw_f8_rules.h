// Which kernels the products of the 8-bit float path take, by their sizes and the device's compute units: plain functions of the host.
#pragma once
#include <math.h>
#include <stdlib.h>
#include <stdint.h>
#include <algorithm>

namespace cw {

constexpr int F8_FEW_WAVES = 8;  // waves of a block of the kernel for few rows

struct F8TileTime {
    int tm, tn;
    double some_b, some_s, all_b, all_s;
};
constexpr F8TileTime F8_TILES[3] = {{64, 64, 2.4, 1.6, 3.0, 1.8}, {128, 128, 4.2, 3.6, 5.5, 4.6}, {256, 256, 12, 9, 15, 13}};
constexpr int64_t F8_MAX_TILES = 1 << 22;  // (a launch holds fewer than 2^32 threads, 512 of a tile at most)
// (-1: every tile's count exceeds the launch)
inline int f8_pick_tile(int64_t m, int64_t n, int rb, int cus) {
    int best = -1;
    double least = 0;
    for (int i = 0; i < 3; i++) {
        const F8TileTime &t = F8_TILES[i];
        const int64_t blocks = (m + t.tm - 1) / t.tm * ((n + t.tn - 1) / t.tn);
        if (blocks >= F8_MAX_TILES) continue;
        const double k = rb / 1024.0, us = (double)(blocks / cus) * (t.all_b + t.all_s * k) + (blocks % cus ? t.some_b + t.some_s * k : 0.0);
        if (best < 0 || us < least) {
            best = i;
            least = us;
        }
    }
    return best;
}
// Groups of 16 rows of x that k_f8_few takes (0: tiles).
inline int f8_few_groups(int64_t m, int64_t n, int rb) {
    if (getenv("FEW")) { int f = atoi(getenv("FEW")); if (!f || m > 128) return 0; int g = (int)((m + 15) / 16); return g == 7 ? 8 : g; }
    return m <= 16 ? 1 : m <= 32 && n * rb <= 1 << 24 ? 2 : m <= 64 && n * rb <= 1 << 21 ? 4 : 0;
}

// Four groups of weight rows a wave instead of two (whose steps are twice as wide and whose sums leave more registers): where the weights'
// bytes bound, at up to 128 picks an expert, and there is a block for every CU twice. Measured in a graph, two / four groups, bf16: 128 experts of
// 2,880 x 2,880, 64 tokens of 4 picks 239 / 202 us, 2,048 tokens (64 an expert) 318 / 275; 256 of 512 x 2,048, 512 of 8 (16) 57 / 51; 64 of
// 1,408 x 2,048, 2,048 of 6 (192) 118 / 125; 8 of 4,096 x 2,048, 2,048 of 2 (512) 115 / 130; 256 of 1,024 x 2,048, 8 of 8 (228 blocks) 28 / 32.
inline bool f8_four_groups(int E, int64_t picks, int64_t n, int cus) {
    const double used = E * (1 - pow(1 - 1.0 / E, (double)picks));
    return picks <= 128ll * E && used * ((n + 255) / 256) >= 2 * cus;
}

}  // namespace cw
