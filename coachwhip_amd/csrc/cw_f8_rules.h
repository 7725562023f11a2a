// Which kernels the products and layers of the 8-bit float path take, by their sizes and the device's compute units: plain functions of the host.
#pragma once
#include <math.h>
#include <stdint.h>
#include <algorithm>

namespace cw {

constexpr int F8_FEW_WAVES = 8;  // waves of a block of the kernel for few rows

// The tile whose estimated time is the least. A CU runs one block of any of them; a round of blocks on every CU takes b + s k / 1024 us, more than
// one on some of them. Exact products (results in f32 and f16) take about twice the time. Measured in a graph (4096 x 4096 in bf16; launch 2.5 us
// included), estimate / measured: 64 x 64 at 128 rows 13.4 / 13.4, 256 rows (every CU) 14.3 / 14.3, 512 rows 26.1 / 29; 128 x 128 at 512 rows 26.9 / 26.9,
// 1,024 rows 29.4 / 29.4, 2,048 rows 56.3 / 55.8; 256 x 256 at 2,048 rows 58.5 / 59.4, 4,096 rows 71.5 / 71.1. In f32: 64 x 64 at 77 rows of 4001 x
// 2880 13.1 / 13.2; 128 x 128 at 512 rows of 4096 x 4096 44 / 44.5; 256 x 256 118 / 118.7.
struct F8TileTime {
    int tm, tn;
    double some_b, some_s, all_b, all_s;
};
constexpr F8TileTime F8_TILES[2][3] = {{{64, 64, 2.6, 2.07, 3.0, 2.2}, {128, 128, 2.8, 5.4, 3.3, 5.9}, {256, 256, 8, 12, 19, 12.5}},
                                       {{64, 64, 2.0, 3.0, 2.4, 3.2}, {128, 128, 1.0, 10.1, 2.0, 11}, {256, 256, 2, 28.4, 4, 30}}};
constexpr int64_t F8_MAX_TILES = 1 << 22;  // (a launch holds fewer than 2^32 threads, 512 of a tile at most)
// (-1: every tile's count exceeds the launch)
inline int f8_pick_tile(bool exact, int64_t m, int64_t n, int rb, int cus) {
    int best = -1;
    double least = 0;
    for (int i = 0; i < 3; i++) {
        const F8TileTime &t = F8_TILES[exact][i];
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
// Groups of 16 rows of x that k_f8_few takes (0: tiles): each block, of 16 columns, reads all of x. Measured in a graph, few rows / 64 x 64 tiles, bf16: 32
// rows of 4096 x 4096 9.1 / 13.4 us, of 8192 x 8192 25.5 / 31; 48 rows of 4096 x 4096 12.6 / 13.4, of 8192 x 8192 34.8 / 31; 64 rows of 2048 x 2048 8.5 /
// 8.7, of 4096 x 4096 15.0 / 13.4. f32, 77 rows: of 4001 x 2880 12.2 / 13.2, of 4096 x 4096 17.7 / 18, of 8192 x 8192 48.5 / 44.
inline int f8_few_groups(bool exact, int64_t m, int64_t n, int cus) {
    const int64_t columns = 16ll * cus;  // a block to a CU
    const int most = exact && n <= columns ? 5 : n <= columns / 2 ? 4 : n <= columns ? 3 : 2;
    return m <= 16 * most ? (int)((m + 15) / 16) : 0;
}

// Four groups of weight rows a wave instead of two (whose steps are twice as wide and whose sums leave more registers): where both the weights' bytes
// and the products count, and there is a block for every CU twice. A long k ends that
// at 64 picks. Measured in a graph, two / four groups, bf16: 128 experts of 2,880 x 2,880, 2 picks each 178 / 190 us, 32 230 / 218, 64 259 / 246, 68 263 / 250, 72 265 / 260, 80
// 274 / 280, 94 291 / 316, 128 360 / 358 to 389 (a k of 2,560: 80 249 / 256; 2,304: 64 212 / 201, 80 225 / 222, 100 244 / 251: the line at 64 gives away 5 % up to 75); 256 of 512 x 2,048 (16) 47.1 / 45.6, (64) 66.8 / 56.9; 256 of 1,024 x 2,048 (64) 136 / 125; 256 of 2,048 x 512
// (16) 65.0 / 52.3, (128) 131 / 120, (192) 177 / 156, of 512 x 2,048 (256) 179 / 171. Exact sums: 128 of 2,880 x 2,880 (64) 326 / 319, (128)
// 543 / 622. With fewer blocks: 64 of 1,408 x 2,048 (192) 100 / 132; 8 of 4,096 x 2,048 (512) 90 / 123.
inline bool f8_four_groups(int E, int64_t picks, int64_t n, int64_t k, int cus) {
    return picks >= 32ll * E && picks <= (k > 2048 ? 64ll : 128ll) * E && E * ((n + 255) / 256) >= 2 * cus;
}
// Few experts of many picks: tiles of 128 sorted rows x 128 of W, one workgroup a CU, whose eight waves share every code through LDS (the kernel of two
// groups reads each expert's rows once for 32 of W). With more than three blocks of W to a CU the two workgroups that the other kernel keeps there hide
// more. Measured in a graph, two groups / tiles, bf16: 8 experts of 4,096 x 2,048, 32 picks each 17.4 / 19.3 us, 64 23.6 / 19.9, 256 57.0 / 48.5,
// 512 90.4 / 80.7, 2,048 256 / 259; 16 of 512 x 4,096 (256) 49.3 / 27.2; 32 of 2,048 x 2,048 (256) 84.1 / 74.7; 64 of 1,408 x 2,048 (64) 45.6 / 47.7,
// (96) 59.5 / 50.9, (384) 158 / 154; 128 of 1,024 x 1,024, four blocks to a CU (64) 36.9 / 44.2, (128) 62.0 / 63.2; 128 of 2,880 x 2,880 (192) 456 / 506.
// Exact sums: 8 of 4,096 x 2,048 (64) 30.7 / 28.1, (128) 59.6 / 53.1, (512) 140 / 116; 64 of 1,408 x 2,048 (64) 62.8 / 71.9, (384) 265 / 253.
inline bool f8_sorted_tiles(bool exact, int E, int64_t picks, int64_t n, int cus) {
    return picks >= (exact ? 128ll : 64ll) * E && E * ((n + 127) / 128) <= 3 * cus;
}

// ------------------------------------------------------------------------------ layers

// Whether a layer takes two launches, which read an expert once for each pick, or the sort and the grouped products, six launches, which
// read it once for its picks. Estimates in us, for their difference: two launches 7 and for each pick the larger of its expert's bytes at 6.5
// TB/s and 4.5 ns for each of its blocks (16 columns of gate and up; 16 outputs of down, which a token's picks share); grouped 26 and the bytes of
// E (1 - (1 - K / E)^T) experts, as many as T tokens pick on average, at 7 TB/s. Measured in a graph that goes round over layers of 1.2 GB or 16, bf16, two
// launches / grouped: 256 experts of 512 x 2,048, top-8, 1 token 12.5 / 36.5, 8 tokens 42 / 57, 20 85 / 93, 24 99 / 113 (which it has grouped), 32
// 126 / 122, 48 182 / 152; 128 of 2,880 x 2,880, top-4, 4 tokens 88 / 104, 5 111 / 109, 8 161 / 152, 16 312 / 245; 8 of 4,096 x 2,048, top-2, 4 40 / 53, 6 54 / 56, 8 68 / 58;
// 64 of 1,408 x 2,048, top-6, 6 70 / 76, 8 89 / 83, 12 128 / 89; 16 of 2,880 x 4,096, top-2, 4 66 / 71, 6 95 / 89; 256 of 1,024 x 4,096, top-8, 4 81 / 85, 8 153 / 151;
// small experts, whose blocks count: 64 of 256 x 1,024, top-8, 24 33 / 36, 32 41 / 36; 16 of 200 x 256, top-4, 48 22 / 24, 64 28 / 24; 64 of 512 x 512, top-1, 64
// 24 / 27, 256 75 / 29. Results in f32 the same but for wide experts, 10 % more in two launches (128 of 2,880 x 2,880, 5 tokens 122 / 112). Over all sizes
// measured it loses 0.4 % to the better of both, 15 % at most.
// The two launches hold a row of x in 32 steps of 128 codes and the K hidden rows in 16 KB of codes: layers beyond that (hidden above 4,096) are
// grouped for any number of tokens.
constexpr int F8_FEW_HIDDEN = 4096, F8_FEW_CODES = 16384;
inline bool f8_few_tokens(int E_, int K_, int H, int I, int T) {
    const int64_t rbh = (H + 127) / 128 * 128, rbi = (I + 127) / 128 * 128;
    if (rbh > F8_FEW_HIDDEN || K_ * rbi > F8_FEW_CODES || T > 1024) return false;
    const double K = K_, E = E_, bytes = 2.0 * I * rbh + (double)H * rbi, blocks = (I + 15) / 16 + (H + 15) / 16 / K;
    return 7 + T * K * std::max(bytes / 6.5e6, 4.5e-3 * blocks) <= 26 + E * (1 - pow(1 - K / E, T)) * bytes / 7e6;
}

}  // namespace cw
