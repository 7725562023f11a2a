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

// A block of WAVES waves, MB blocks of 16 activation rows shared by all of them, NW groups of 16 weight rows for
// each wave. The activations go through a ring of three LDS stages of 16 MB rows x 128 bytes (direct
// global-to-LDS loads, two steps ahead, one barrier a step); a wave's weights, which no other wave reads, come
// straight into its registers one step ahead. Chunk c (16 bytes) of row r lies at chunk c ^ (r & 7) of its LDS
// row, which the loading lane's global address does: eight rows' reads of one chunk touch all banks once.
template <int MB, int WAVES>
struct I8Stage {
    static constexpr int ROWS = 16 * MB, BYTES = ROWS * I8_STEP, LDS = 3 * BYTES;
    static constexpr int LOADS = 2 * MB;                        // of 1,024 bytes each, a stage
    static constexpr int PER = (LOADS + WAVES - 1) / WAVES;     // of a wave
};

// xrow(r): the first byte of activation row r < 16 MB of the tile (any valid row past its end); wrow[j]: that of
// the lane's weight row of group j, + 16 (lane / 16)
template <int MB, int NW, int WAVES, class XRow>
__device__ __forceinline__ void i8_loop(uint8_t *lds, XRow xrow, const uint8_t *const (&wrow)[NW], int steps, i32x4 (&acc)[MB][NW]) {
    using S = I8Stage<MB, WAVES>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint8_t *xp[S::PER];
    uint32_t to[S::PER];
#pragma unroll
    for (int i = 0; i < S::PER; i++) {
        const int r = 8 * (wave + WAVES * i) + (lane >> 3);
        xp[i] = xrow(r < S::ROWS ? r : S::ROWS - 1) + 16 * ((lane & 7) ^ (r & 7));
        to[i] = lds_addr(lds) + 1024 * (wave + WAVES * i);
    }
    auto fetch_x = [&](int step) __attribute__((always_inline)) {
        const uint32_t stage = (step % 3) * S::BYTES;
#pragma unroll
        for (int i = 0; i < S::PER; i++)
            if (S::LOADS % WAVES == 0 || wave + WAVES * i < S::LOADS) dma16(xp[i] + (int64_t)step * I8_STEP, __builtin_amdgcn_readfirstlane(to[i] + stage));
    };
    i32x4 w[2][NW][2];
    auto fetch_w = [&](int step, i32x4 (&v)[NW][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NW; j++) {
            v[j][0] = load16(wrow[j] + (int64_t)step * I8_STEP);
            v[j][1] = load16(wrow[j] + (int64_t)step * I8_STEP + 64);
        }
    };
    auto multiply = [&](int step, const i32x4 (&v)[NW][2]) __attribute__((always_inline)) {
        const uint8_t *b = lds + (step % 3) * S::BYTES + (lane & 15) * I8_STEP;
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
            for (int mb = 0; mb < MB; mb++) {
                const i32x4 x = *(const i32x4 *)(b + mb * 16 * I8_STEP + 16 * ((4 * kk + (lane >> 4)) ^ (lane & 7)));
#pragma unroll
                for (int j = 0; j < NW; j++) acc[mb][j] = mfma_i8(v[j][kk], x, acc[mb][j]);
            }
    };
    // the stage of `step` is in LDS for every wave, and every wave is done with the stage before it. (Loads return
    // in order: this wave's older ones, its part of the stage among them, are in when the weights of the step,
    // which it waits for anyway, are.)
    auto ready = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int j = 0; j < NW; j++) acc[mb][j] = i32x4{0, 0, 0, 0};
    fetch_x(0);
    fetch_w(0, w[0]);
    for (int step = 0; step < steps; step += 2) {
        ready();
        if (step + 1 < steps) {
            fetch_x(step + 1);
            fetch_w(step + 1, w[1]);
        }
        multiply(step, w[0]);
        if (step + 1 >= steps) break;
        ready();
        if (step + 2 < steps) {
            fetch_x(step + 2);
            fetch_w(step + 2, w[0]);
        }
        multiply(step + 1, w[1]);
    }
}

}  // namespace cw
