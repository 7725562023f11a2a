// The product of a block's rows of 8-bit activations with 8-bit weight rows on the matrix cores.
#pragma once
#include "cw_gmm_dev.h"
#include "cw_i8_dev.h"

namespace cw {

// v_mfma_i32_16x16x64_i8: lane l gives 16 codes of weight row l % 16 (A) and of activation row l % 16 (B), both
// from 16 (l / 16) of the 64 of the step (any order of k is right that both operands share), and holds weight
// rows 4 (l / 16) + 0..3 of activation row l % 16 of the 16 x 16 sums: four neighbouring outputs of one row.
__device__ __forceinline__ i32x4 mfma_i8(i32x4 w, i32x4 x, i32x4 acc) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, acc, 0, 0, 0); }

__device__ __forceinline__ i32x4 load16(const uint8_t *p) { return *(const i32x4 *)p; }

constexpr int I8_STEP = 128;  // codes of k per step: whole cache lines of every row

// A block of four waves over a stream of weights: MB blocks of 16 activation rows shared by all of them, NW groups of
// 16 weight rows for each wave, k in steps of 512 / NW codes (NW 2: 256, where the weights' bytes bound; NW 4: 128,
// half the reads of LDS for a product, where many rows share the weights). A wave's weights, which no other wave reads,
// come straight into its registers, a whole step ahead: the step's neighbouring bytes of a row asked for together. The
// activations go through registers (two steps ahead) into two LDS stages of 16 MB rows, one barrier a step; chunk c (16
// bytes) of row r lies at chunk c ^ (r % chunks of a row) of its LDS row: the reads of one chunk touch all banks once.
template <int MB, int NW>
struct I8Stage {
    static constexpr int WIDE = 512 / NW, CHUNKS = WIDE / 16, BYTES = 16 * MB * WIDE, LDS = 2 * BYTES;
    static constexpr int ROWS = 64 / CHUNKS, LOADS = 16 * MB / ROWS, PER = (LOADS + 3) / 4;  // rows of a load, loads of a stage and of a wave
};

// x0 and w0 (NW / MATS groups each): wave-uniform, 4 GiB at most below any row used; xrow(r): the offset from x0 of
// activation row r < 16 MB of the tile (any valid row past its end); wrow[j]: that from w0 of the lane's weight
// row of group j, + 16 (lane / 16); rb: bytes of a row, a multiple of 128
template <int MB, int NW, int MATS, class XRow>
__device__ __forceinline__ void i8_loop(uint8_t *lds, const uint8_t *x0, XRow xrow, const uint8_t *const (&w0)[MATS], const uint32_t (&wrow)[NW], int rb,
                                        i32x4 (&acc)[MB][NW]) {
    using S = I8Stage<MB, NW>;
    constexpr int WIDE = S::WIDE, Q = WIDE / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = (rb + WIDE - 1) / WIDE, chunk = lane % S::CHUNKS;
    // load i of this wave: the rows from ROWS (wave + 4 i) (with fewer loads than waves, some twice: the same bytes to
    // the same place)
    uint32_t xp[S::PER];
    int xl[S::PER];
#pragma unroll
    for (int i = 0; i < S::PER; i++) {
        const int r = S::ROWS * ((wave + 4 * i) % S::LOADS) + lane / S::CHUNKS;
        xp[i] = xrow(r);
        xl[i] = r * WIDE + 16 * (chunk ^ (r % S::CHUNKS));
    }
    i32x4 xr[S::PER], w[2][NW][Q];
    // the lane's chunk of k of a step, and whether the row has it (past its end: its last line, not used)
    auto fetch_x = [&](int step) __attribute__((always_inline)) {
        const int o = min(step * WIDE + 16 * chunk, rb - 16);
#pragma unroll
        for (int i = 0; i < S::PER; i++) xr[i] = load16(x0 + (xp[i] + (uint32_t)o));
    };
    auto store_x = [&](int step) __attribute__((always_inline)) {
        const bool in = step * WIDE + 16 * chunk < rb;
        uint8_t *to = lds + (step & 1) * S::BYTES;
#pragma unroll
        for (int i = 0; i < S::PER; i++) *(i32x4 *)(to + xl[i]) = in ? xr[i] : i32x4{0, 0, 0, 0};
    };
    auto fetch_w = [&](int step, i32x4 (&v)[NW][Q]) __attribute__((always_inline)) {
        const int o = min(step * WIDE, rb - 128), o2 = min(step * WIDE + 128, rb - 128);
#pragma unroll
        for (int j = 0; j < NW; j++) {
            const uint8_t *b = w0[j / (NW / MATS)];
            v[j][0] = load16(b + o + wrow[j]);
            v[j][1] = load16(b + o + 64 + wrow[j]);
            if constexpr (Q == 4) {
                v[j][2] = load16(b + o2 + wrow[j]);
                v[j][3] = load16(b + o2 + 64 + wrow[j]);
            }
        }
    };
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int j = 0; j < NW; j++) acc[mb][j] = i32x4{0, 0, 0, 0};
    auto body = [&](int step, i32x4 (&now)[NW][Q], i32x4 (&next)[NW][Q]) __attribute__((always_inline)) {
        // every wave's part of the stage is in LDS, and every wave has multiplied the stage before it, whose buffer
        // the next one takes
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        store_x(step + 1);
        __builtin_amdgcn_sched_barrier(0);
        fetch_x(step + 2);
        fetch_w(step + 1, next);
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t *b = lds + (step & 1) * S::BYTES + (lane & 15) * WIDE;
        auto frag = [&](int f) __attribute__((always_inline)) {
            return *(const i32x4 *)(b + (f % MB) * 16 * WIDE + 16 * ((4 * (f / MB) + (lane >> 4)) ^ (lane & (S::CHUNKS - 1))));
        };
        i32x4 x = frag(0);
#pragma unroll
        for (int f = 0; f < Q * MB; f++) {
            // the next fragment of x is read while this one is multiplied (the fences keep the compiler from reading
            // them all at once)
            i32x4 xn = x;
            if (f + 1 < Q * MB) xn = frag(f + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NW; j++) acc[f % MB][j] = mfma_i8(now[j][f / MB], x, acc[f % MB][j]);
            __builtin_amdgcn_sched_barrier(0);
            x = xn;
        }
    };
    fetch_x(0);
    store_x(0);
    fetch_x(1);
    __builtin_amdgcn_sched_barrier(0);
    fetch_w(0, w[0]);
    for (int step = 0; step < steps; step += 2) {  // (a step past the end multiplies zeros)
        body(step, w[0], w[1]);
        body(step + 1, w[1], w[0]);
    }
}

}  // namespace cw
