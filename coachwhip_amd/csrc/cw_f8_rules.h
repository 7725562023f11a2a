// Which kernels the products of the 8-bit float path take, by their sizes and the device's compute units: plain functions of the host.
#pragma once
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
    return m <= 16 ? 1 : m <= 32 && n * rb <= 1 << 24 ? 2 : m <= 64 && n * rb <= 1 << 21 ? 4 : 0;
}

}  // namespace cw
