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
// each wave. The activations go through registers (two steps ahead) into two LDS stages of 16 MB rows x 128 bytes,
// one barrier a step; a wave's weights, which no other wave reads, come straight into its registers, each half of
// a step's loaded as soon as that of the step before is used up. Chunk c (16 bytes) of row r lies at chunk
// c ^ (r & 7) of its LDS row: eight rows' reads of one chunk touch all banks once.
template <int MB, int WAVES>
struct I8Stage {
    static constexpr int ROWS = 16 * MB, BYTES = ROWS * I8_STEP, LDS = 2 * BYTES;
    static constexpr int LOADS = 2 * MB;                        // of 1,024 bytes each, a stage
    static constexpr int PER = (LOADS + WAVES - 1) / WAVES;     // of a wave
};

// x0 and w0 (NW / MATS groups each): wave-uniform, 4 GiB at most below any row used; xrow(r): the offset from x0 of
// activation row r < 16 MB of the tile (any valid row past its end); wrow[j]: that from w0 of the lane's weight
// row of group j, + 16 (lane / 16)
template <int MB, int NW, int WAVES, int MATS, class XRow>
__device__ __forceinline__ void i8_loop(uint8_t *lds, const uint8_t *x0, XRow xrow, const uint8_t *const (&w0)[MATS], const uint32_t (&wrow)[NW], int steps,
                                        i32x4 (&acc)[MB][NW]) {
    using S = I8Stage<MB, WAVES>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t xp[S::PER];
#pragma unroll
    for (int i = 0; i < S::PER; i++) {
        // (with fewer loads than waves some waves copy the same rows: the same bytes to the same place)
        const int r = 8 * ((wave + WAVES * i) % S::LOADS) + (lane >> 3);
        xp[i] = xrow(r) + 16 * ((lane & 7) ^ (r & 7));
    }
    i32x4 xr[S::PER];
    auto fetch_x = [&](int step) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < S::PER; i++) xr[i] = load16(x0 + (int64_t)step * I8_STEP + xp[i]);
    };
    auto store_x = [&](int step) __attribute__((always_inline)) {
        uint8_t *at = lds + (step & 1) * S::BYTES + 16 * lane;
#pragma unroll
        for (int i = 0; i < S::PER; i++) *(i32x4 *)(at + 1024 * ((wave + WAVES * i) % S::LOADS)) = xr[i];
    };
    i32x4 w[2][NW];  // both halves of a step's 128 codes of k
    auto fetch_w = [&](int step, int kk) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NW; j++) w[kk][j] = load16(w0[j / (NW / MATS)] + (int64_t)step * I8_STEP + wrow[j] + 64 * kk);
    };
    const uint32_t xl = (lane & 15) * I8_STEP;
    const int c[2] = {16 * ((lane >> 4) ^ (lane & 7)), 16 * ((4 + (lane >> 4)) ^ (lane & 7))};
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int j = 0; j < NW; j++) acc[mb][j] = i32x4{0, 0, 0, 0};
    const int last = steps - 1;  // (loads past it repeat it, unused)
    fetch_x(0);
    store_x(0);
    // (in the order of the loop, from which the compiler counts how many loads a wait may leave open)
    fetch_x(min(1, last));
    __builtin_amdgcn_sched_barrier(0);
    fetch_w(0, 0);
    __builtin_amdgcn_sched_barrier(0);
    fetch_w(0, 1);
    __builtin_amdgcn_sched_barrier(0);
    for (int step = 0; step < steps; step++) {
        // every wave's part of the stage is in LDS, and every wave has multiplied the stage before it, whose buffer
        // the next one takes
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        store_x(step + 1);
        __builtin_amdgcn_sched_barrier(0);
        fetch_x(min(step + 2, last));
        const uint8_t *b = lds + (step & 1) * S::BYTES + xl;
        i32x4 x = *(const i32x4 *)(b + c[0]);
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
#pragma unroll
            for (int mb = 0; mb < MB; mb++) {
                // the next fragment of x is read while this one is multiplied; the fences keep the compiler from reading
                // them all at once, and the weights of the next step before this one's are used up: there are no
                // registers for that
                const int f = kk * MB + mb + 1;
                i32x4 xn = x;
                if (f < 2 * MB) xn = *(const i32x4 *)(b + (f % MB) * 16 * I8_STEP + c[f / MB]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < NW; j++) acc[mb][j] = mfma_i8(w[kk][j], x, acc[mb][j]);
                __builtin_amdgcn_sched_barrier(0);
                x = xn;
            }
            fetch_w(min(step + 1, last), kk);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

}  // namespace cw
