// Which kernels the products and layers of the 8-bit integer path take, by their sizes and the device's compute units: plain
// functions of the host, each with what was measured on both sides of its lines.
#pragma once
#include <math.h>
#include <stdint.h>
#include <algorithm>

namespace cw {

// ------------------------------------------------------------------------------ products

constexpr int I8_FEW_WAVES = 8;  // waves of a block of the kernels for few rows and few tokens

// The tile whose estimated time is the least. A CU runs one block of any of them; a round of blocks on every CU takes
// b + s k / 1024 us, more than one on some of them (whose share of L2 and of the fabric is larger). Measured in a graph (4096 x
// 4096 in bf16; launch 2.5 us included), estimate / measured: 64 x 64 at 128 rows 10.7 / 11.3, 256 rows (every CU) 11.9 / 11.8,
// 512 rows 21.3 / 23.0; 64 x 128 at 256 rows 14.5 / 15.3, 512 rows 16.1 / 16.4, 1,024 rows 29.7 / 29.7; 128 x 128 at
// 512 rows 19.5 / 22.2, 1,024 rows 25.2 / 23.6, 2,048 rows 47.9 / 46.5, 4,096 rows 93.3 / 89.3; 256 x 256 at 2,048 rows 46.5 /
// 52.0, 4,096 rows 65.1 / 60.3, 8,192 rows 128 / 120. So the estimates are off by up to a tenth, and at 2,048 rows of that
// matrix the slower tile is taken (52.0 instead of 46.5).
struct I8TileTime {
    int tm, tn;
    double some_b, some_s, all_b, all_s;
};
constexpr I8TileTime I8_TILES[4] = {{64, 64, 2.4, 1.45, 3.0, 1.6}, {64, 128, 3.4, 2.15, 4.0, 2.4}, {128, 128, 4.2, 3.2, 5.5, 4.3}, {256, 256, 12, 8, 15, 11.9}};
constexpr int64_t I8_MAX_TILES = 1 << 22;  // (a launch holds fewer than 2^32 threads, 512 of a tile at most)
// (-1: every tile's count exceeds the launch)
inline int i8_pick_tile(int64_t m, int64_t n, int rb, int cus) {
    int best = -1;
    double least = 0;
    for (int i = 0; i < 4; i++) {
        const I8TileTime &t = I8_TILES[i];
        const int64_t blocks = (m + t.tm - 1) / t.tm * ((n + t.tn - 1) / t.tn);
        if (blocks >= I8_MAX_TILES) continue;
        const double k = rb / 1024.0, us = (double)(blocks / cus) * (t.all_b + t.all_s * k) + (blocks % cus ? t.some_b + t.some_s * k : 0.0);
        if (best < 0 || us < least) {
            best = i;
            least = us;
        }
    }
    return best;
}
// Groups of 16 rows of x that k_i8_few takes (0: tiles). Measured in a graph, few rows / 64 x 64 tiles: 16 rows of 4096 x 4096
// 6.6 / 10.1 us, of 8192 x 8192 18.9 / 17.9; 32 rows 8.8 / 10.8 and 26.3 / 20.2 (each block reads all of x); 64 rows of 1024 x 1024
// 4.9 / 5.7, of 2048 x 2048 7.2 / 7.2.
inline int i8_few_groups(int64_t m, int64_t n, int rb) {
    return m <= 16 ? 1 : m <= 32 && n * rb <= 1 << 24 ? 2 : m <= 64 && n * rb <= 1 << 21 ? 4 : 0;
}

// ------------------------------------------------------------------------------ layers

constexpr int I8_TILE = 128;        // picks of a tile, at most
constexpr int I8_PLAN_TOKENS = 32;  // tokens that the plan routes itself

inline int64_t i8_max_tiles(int64_t picks, int experts) { return (picks + I8_TILE - 1) / I8_TILE + std::min<int64_t>(experts, picks); }
// logits of a lane in the routing
inline int i8_route_width(int E) { return E <= 256 ? 4 : E <= 512 ? 8 : 16; }

// Two launches read an expert once per pick, the grouped ones once per tile: about 15 us more for their launches, but
// each byte once. The picks' reads beyond the distinct experts', E (1 - (1 - K / E)^T) on average, come in part from the
// caches. Measured in a graph, two launches / grouped, and those bytes: 256 experts of 512 x 2,048, top-8, 16 tokens 69 / 97 us
// (82 MB), 32 tokens 121 / 136 (292); 128 of 2,880 x 2,880, top-4, 6 tokens 123 / 137 (46), 8 tokens 157 / 175 (84),
// 16 tokens 290 / 264 (331); 8 of 2,048 x 4,096, top-2, 6 tokens 42 / 46 (137), 8 tokens 52 / 51 (222); 512 of 512 x
// 2,048, top-10, 32 tokens 180 / 182 (253). Bytes alone do not decide: 32 tokens over the 256 small experts take the slower form.
// The two launches hold a row of x in four pieces a lane and the K hidden rows in 16 KB: layers beyond that (hidden above 4,096;
// top-2 with an inter of 14,336 and hidden 4,096: 118 us for one token, of 69 for its bytes) are grouped for any number of tokens.
inline bool i8_few_tokens(int E_, int K_, int H, int I, int T) {
    const int64_t rbh = (H + 127) / 128 * 128, rbi = (I + 127) / 128 * 128;
    if (rbh > 4 * 1024 || K_ * rbi > 16 * 1024 || T > 1024) return false;
    const double K = K_, E = E_, picks = T * K, distinct = E * (1 - pow(1 - K / E, T));
    return (picks - distinct) * (2.0 * I * rbh + (double)H * rbi) <= 200e6;
}

// The kernels of a few tokens: pieces of 16 bytes that a lane holds of a row of x (gate and up) or of the K hidden rows end to end
// (down), and rows of weights a wave: more where that still leaves every CU four blocks (the routing and the rows' codes are made
// once a block).
inline int i8_gateup_pieces(int rbh) { return (rbh + 1023) / 1024; }
inline int i8_gateup_rows(int pieces, int I, int64_t picks, int cus) {
    const int64_t blocks = (I + I8_FEW_WAVES - 1) / I8_FEW_WAVES * picks;
    return pieces <= 2 && blocks >= 16 * cus ? 4 : blocks >= 2 * cus ? 2 : 1;
}
inline int i8_down_pieces(int K, int rbi) {
    const int pieces = (K * (rbi / 16) + 63) / 64;
    return pieces <= 2 ? pieces : pieces <= 4 ? 4 : pieces <= 8 ? 8 : pieces <= 12 ? 12 : 16;
}
inline int i8_down_rows(int pieces, int H, int64_t T, int cus) {
    const int64_t blocks = (H + I8_FEW_WAVES - 1) / I8_FEW_WAVES * T;
    return pieces <= 4 && blocks >= 16 * cus ? 4 : pieces <= 8 && blocks >= 8 * cus ? 2 : 1;
}

// Four groups of weight rows a wave instead of two, where the picks share the weights and there are blocks for every CU
// twice. Measured in a graph, two / four groups: 128 experts of 2,880 x 2,880, top-4, 64 tokens (2 picks an expert) 533 / 551 us,
// 512 tokens (16) 670 / 667, 2,048 tokens (64) 821 / 788; 256 of 512 x 2,048, top-8, 512 tokens (16) 212 / 200; 64 of
// 1,408 x 2,048, top-6, 2,048 tokens (192) 306 / 273; 16 of 2,880 x 4,096, top-2, 512 tokens (64, 368 blocks) 168 / 177,
// 2,048 tokens (256, 736 blocks) 346 / 312.
inline bool i8_many_picks(int E, int K, int I, int T, int cus) {
    const double avg = (double)T * K / E;
    return avg >= 12 && E * ceil(avg / I8_TILE) * ((I + 127) / 128) >= 2 * cus;
}

}  // namespace cw
