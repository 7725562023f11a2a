// Products of rows of e4m3 codes with e4m3 matrices, scales of 128 columns of k (gfx950): one matrix, or of sorted rows each with its
// expert's.
#include <atomic>

#include "cw_f8_rules.h"
#include "cw_f8_tile.h"
#include "cw_mfma.h"
#include "cw_piles.h"

namespace cw {

struct F8MatArgs {
    const uint8_t *w, *x;
    const float *ws, *xs, *bias;
    int64_t n, m;    // m: rows of x, whose scales are m apart
    int rb, blocks;  // bytes of a row, scales of a row
    void *y;
    int64_t ldy;
    // sorted rows
    int64_t w_stride, ws_stride;  // from an expert's to the next
    const void *tiles;
    const int *order;  // NULL: x holds the sorted rows; else x's row of a position is order / K
    int K, E;
};

// Few rows of x: a block takes 16 rows of W and up to 16 MB of x over all of k, its waves the steps of 128 codes in turn, both
// operands straight from memory into registers (no byte of either is used by two waves of a block). The waves' sums meet in LDS: the
// upper four's onto the lower four's, then those in their order. One row of 2048 x 2048: 4.0 us, a launch, one round trip and the join; 77 rows of 4001 x 2880 in
// f32 12.2 in a graph: each block makes x's codes f16 for itself.
template <class T, int MB, bool EXACT>
__global__ __launch_bounds__(64 * F8_FEW_WAVES) void k_f8_few(F8MatArgs a) {
    constexpr int HALF = F8_FEW_WAVES / 2;
    __shared__ f32x4 part[HALF][MB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = 16 * (lane >> 4);
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const uint8_t *w0 = a.w + n0 * a.rb;
    const float *ws = f8_uniform(a.ws + n0 / F8_BLOCK * a.blocks);
    const uint32_t wrow = (uint32_t)(min(lane & 15, (int)(a.n - 1 - n0)) * a.rb + at);
    uint32_t xrow[MB], srow[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) {
        srow[i] = min(16 * i + (lane & 15), (int)a.m - 1);
        xrow[i] = srow[i] * a.rb + at;
    }
    f32x4 acc[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    bool strange = false;
    for (int step = wave; step < a.blocks; step += F8_FEW_WAVES) {
        const uint8_t *w = w0 + (int64_t)step * F8_BLOCK + wrow, *x = a.x + (int64_t)step * F8_BLOCK;
        F8Frag<EXACT> wf, xf;
        wf.load(w, w + 64);
        const float sw = f8_scale_at(ws + step);
        strange |= f8_strange(sw);
        float sx[MB];
#pragma unroll
        for (int i = 0; i < MB; i++) {
            sx[i] = a.xs[step * a.m + srow[i]];
            if (i % 4 == lane >> 4) strange |= f8_strange(sx[i]);
        }
#pragma unroll
        for (int i = 0; i < MB; i++) {
            xf.load(x + xrow[i], x + xrow[i] + 64);
            const f32x4 p = F8Frag<EXACT>::product(wf, xf);
#pragma unroll
            for (int c = 0; c < 4; c++) acc[i][c] = fmaf(p[c], sx[i] * sw, acc[i][c]);
        }
    }
    if (wave >= HALF)
#pragma unroll
        for (int i = 0; i < MB; i++) part[wave - HALF][i][lane] = acc[i];
    strange = __syncthreads_or(strange);
    if (wave < HALF)
#pragma unroll
        for (int i = 0; i < MB; i++) part[wave][i][lane] += acc[i];
    __syncthreads();
    const int64_t m = 16 * wave + (lane & 15), n = n0 + 4 * (lane >> 4);
    if (wave >= MB || m >= a.m || n >= a.n) return;
    float b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = a.bias ? a.bias[min(n + i, a.n - 1)] : 0.f;
    f32x4 v = part[0][wave][lane];
#pragma unroll
    for (int o = 1; o < HALF; o++) v += part[o][wave][lane];
    if (strange) f8_strange_sums(a.x + m * a.rb, a.xs + m, a.m, a.w + n * a.rb, ws, a.rb, (int)min(a.n - n, (int64_t)4), v);
    f8_store4((T *)a.y + m * a.ldy + n, (int)min(a.n - n, (int64_t)4), v, b);
}

// Blocks go to the eight dies in turn: each die gets a contiguous range of tiles, in panels of four tiles of W, so that
// those which it runs at once share both operands through its cache.
__device__ __forceinline__ void f8_tile_of_block(int tiles_m, int tiles_n, int tm, int tn, int64_t &m0, int64_t &n0) {
    const int total = tiles_m * tiles_n, die = blockIdx.x & 7, per = total >> 3, rest = total & 7;
    const int id = die * per + min(die, rest) + (int)(blockIdx.x >> 3);
    const int panel = id / (4 * tiles_m), width = min(4, tiles_n - 4 * panel), in = id - panel * 4 * tiles_m;
    m0 = (int64_t)__builtin_amdgcn_readfirstlane(in / width) * tm;
    n0 = (int64_t)__builtin_amdgcn_readfirstlane(4 * panel + in % width) * tn;
}

// A tile of 16 WM MF rows of x by 16 WN NF rows of W, a wave of 16 MF x 16 NF each; codes and scales of Q steps a stage through a ring
// of LDS stages by direct global-to-LDS loads, chunk c (16 bytes) of row r at chunk c ^ (r % 8) of its 128 bytes: the reads of one
// chunk touch all banks once.
template <int WN, int WM, int NF, int MF, int Q, int STAGES>
struct F8Ring {
    static constexpr int TN = 16 * WN * NF, TM = 16 * WM * MF, WAVES = WN * WM, NT = 64 * WAVES;
    static constexpr int CODES = (TN + TM) * F8_BLOCK, STEP = CODES + 4 * TM, STAGE = Q * STEP;
    static constexpr int PER = (TN + TM) / 8 / WAVES, D = STAGES - 1, LDS = STAGES * STAGE;  // loads of codes of a wave and step; stages ahead
    static_assert((TN + TM) % (8 * WAVES) == 0 && TN % (8 * WAVES) == 0 && TM % 64 == 0 && TM / 64 <= WAVES && D * Q * (PER + 1) < 64, "whole loads for every wave");
    static_assert(LDS <= 159 * 1024, "the ring fits the CU");
};
// After a tile's outputs are stored, those with strange scales again: rows m0 .. m_end - 1 of y (x's: xrow), columns n0 .. n0 + cols - 1 of the
// matrix w, ws. (Behind the stores, where no sums are held: beside them this cost the tiles of 256 x 256 registers, and 45 MB of spills.)
template <class T, class XRow>
__device__ __forceinline__ void f8_strange_tile(const F8MatArgs &a, const uint8_t *w, const float *ws, const float *bias, XRow xrow, int64_t m0, int64_t m_end,
                                                int64_t n0, int cols) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const int quads = cols / 4, n = (int)(m_end - m0) * quads;
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int64_t m = m0 + i / quads, c = n0 + 4 * (i % quads);
        if (c >= a.n) continue;
        const int64_t row = xrow(m);
        const int valid = (int)min(a.n - c, (int64_t)4);
        f32x4 v;
        if (!f8_strange_sums(a.x + row * a.rb, a.xs + row, a.m, w + c * a.rb, ws + c / F8_BLOCK * a.blocks, a.rb, valid, v)) continue;
        float b[4];
#pragma unroll
        for (int k = 0; k < 4; k++) b[k] = bias ? bias[min(c + k, a.n - 1)] : 0.f;
        f8_store4((T *)a.y + m * a.ldy + c, valid, v, b);
    }
}
// A wave's sums stored: rows m0.. of m_end of y, columns n0.. . All biases are loaded before the bounds checks, from clamped places. Where all its
// columns are inside, 16 rows at a time go through LDS (`stage`: 16 rows of this wave alone, chunk c of 16 bytes of row r at c ^ (r % chunks)) and
// leave as whole rows, 16 bytes a lane (8,192 sorted rows of 2,880 x 2,880 262 -> 249 us; 8,192 x 4,096 x 4,096 the same either way, of which its
// 67 MB take 12 to 16: all blocks write at once).
template <class T, int MF, int NF>
__device__ __forceinline__ void f8_finish(const F8MatArgs &a, const float *bias, int64_t m0, int64_t m_end, int64_t n0, const f32x4 (&acc)[MF][NF], uint8_t *stage) {
    const int lane = threadIdx.x & 63;
    const int64_t m = m0 + (lane & 15), n = n0 + 4 * (lane >> 4);
    float b[NF][4];
#pragma unroll
    for (int j = 0; j < NF; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) b[j][c] = bias ? bias[min(n + 16 * j + c, a.n - 1)] : 0.f;
    constexpr int ROW = 16 * NF * sizeof(T), CHUNKS = ROW / 16, ROWS = 64 / CHUNKS;  // rows of a store of the wave
    if (n0 + 16 * NF <= a.n) {
#pragma unroll
        for (int i = 0; i < MF; i++) {
            if (m0 + 16 * i >= m_end) break;
#pragma unroll
            for (int j = 0; j < NF; j++) {
                float f[4];
#pragma unroll
                for (int c = 0; c < 4; c++) f[c] = acc[i][j][c] + b[j][c];
                const int r = lane & 15, at = (16 * j + 4 * (lane >> 4)) * (int)sizeof(T);
                store_row<4>((T *)(stage + r * ROW + 16 * ((at / 16) ^ (r & (CHUNKS - 1))) + at % 16), 4, f);
            }
            __builtin_amdgcn_wave_barrier();  // (a wave's reads and writes of LDS are in order)
#pragma unroll
            for (int q = 0; q < (ROWS < 16 ? 16 / ROWS : 1); q++) {
                const int r = ROWS * q + lane / CHUNKS, c = lane % CHUNKS;
                if (r >= 16) break;
                const i32x4 v = *(const i32x4 *)(stage + r * ROW + 16 * (c ^ (r & (CHUNKS - 1))));
                if (m0 + 16 * i + r < m_end) memcpy((uint8_t *)((T *)a.y + (m0 + 16 * i + r) * a.ldy + n0) + 16 * c, &v, 16);
            }
            __builtin_amdgcn_wave_barrier();
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < MF; i++) {
        if (m + 16 * i >= m_end) continue;
#pragma unroll
        for (int j = 0; j < NF; j++)
            if (n + 16 * j < a.n) f8_store4((T *)a.y + (m + 16 * i) * a.ldy + n + 16 * j, (int)min(a.n - n - 16 * j, (int64_t)4), acc[i][j], b[j]);
    }
}

// Whether a tile has a strange scale: its rows' from m0, its weights' from row n0, looked at once, while the first codes are on their way (in the
// steps, where every wave meets them, the checks were a sixth of the instructions).
template <int TM, int TN, int WAVES, class XRow>
__device__ __forceinline__ bool f8_any_strange(const F8MatArgs &a, const float *ws, XRow xrow, int64_t n0) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    bool strange = false;
    const float *xs[TM / 64];
#pragma unroll
    for (int i = 0; i < TM / 64; i++) xs[i] = a.xs + xrow(64 * i + lane);
    for (int b = wave; b < a.blocks; b += WAVES)
#pragma unroll
        for (int i = 0; i < TM / 64; i++) strange |= f8_strange(xs[i][b * a.m]);
    const int64_t last = (a.n - 1) / F8_BLOCK;
#pragma unroll
    for (int c = 0; c < (TN + F8_BLOCK - 1) / F8_BLOCK; c++)
        for (int b = threadIdx.x; b < a.blocks; b += 64 * WAVES) strange |= f8_strange(ws[min(n0 / F8_BLOCK + c, last) * a.blocks + b]);
    return strange;
}
// positions of no expert: zeros
template <class T>
__device__ __forceinline__ void f8_zeros(const F8MatArgs &a, const PileTile &tl, int64_t n0, int cols) {
    const int wide = (int)min(a.n - n0, (int64_t)cols);
    for (int i = threadIdx.x; i < tl.m * wide; i += blockDim.x) ((T *)a.y)[(int64_t)(tl.pos0 + i / wide) * a.ldy + n0 + i % wide] = from_f32<T>(0.f);
}

// SORTED: a tile of sorted rows times their expert's matrix (tiles_n blocks of columns). 4,096 over 8 experts of 4,096 x 2,048 80.7 us (852 TFLOP/s), over 32
// of 2,048 x 2,048 and 8,192 rows 74.7 (920): the chain of a stage, as without sorting.
template <class T, bool EXACT, bool SORTED, int WN, int WM, int NF, int MF, int Q, int STAGES>
__global__ __launch_bounds__(64 * WN *WM, WN *WM / 4) void k_f8_tile(F8MatArgs a, int tiles_m, int tiles_n) {
    using R = F8Ring<WN, WM, NF, MF, Q, STAGES>;
    extern __shared__ __align__(1024) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN;
    const int last = a.blocks - 1, stages = (a.blocks + Q - 1) / Q;
    int64_t m0, n0, m_end = a.m;
    const uint8_t *w = a.w;
    const float *ws = a.ws, *bias = a.bias;
    if constexpr (SORTED) {
        PileTile tl;
        int nb;
        if (!f8_item_of_block(a.tiles, tiles_n, tl, nb)) return;
        n0 = (int64_t)R::TN * nb;
        if (tl.expert == a.E) return f8_zeros<T>(a, tl, n0, R::TN);
        m0 = tl.pos0;
        m_end = tl.pos0 + tl.m;
        w += tl.expert * a.w_stride;
        ws += tl.expert * a.ws_stride;
        if (bias) bias += tl.expert * a.n;
    } else {
        f8_tile_of_block(tiles_m, tiles_n, R::TM, R::TN, m0, n0);
    }
    // x's row of a row of y
    auto row_at = [&](int64_t m) __attribute__((always_inline)) { return SORTED && a.order ? (int64_t)(a.order[m] / a.K) : m; };
    auto xrow = [&](int r) __attribute__((always_inline)) { return row_at(min(m0 + r, m_end - 1)); };
    const uint8_t *w0 = f8_uniform(w + n0 * a.rb), *x0 = a.x + m0 * a.rb;
    // load i of this wave: 8 rows, of TN of W, then TM of x, from 8 (wave + WAVES i); sorted rows of x lie anywhere
    uint32_t off[R::PER];
    const uint8_t *xp[R::PER];
#pragma unroll
    for (int i = 0; i < R::PER; i++) {
        const int r = 8 * (wave + R::WAVES * i) + (lane >> 3), c = 16 * ((lane & 7) ^ (r & 7));
        const bool of_w = 8 * R::WAVES * i < R::TN;
        if (SORTED && !of_w) xp[i] = a.x + xrow(r - R::TN) * a.rb + c;
        else off[i] = (uint32_t)(of_w ? min((int64_t)r, a.n - 1 - n0) : min((int64_t)r - R::TN, a.m - 1 - m0)) * a.rb + c;
    }
    const bool scales = wave < R::TM / 64;  // the waves that load them, 64 each
    const float *xs = a.xs + xrow(min(64 * wave + lane, R::TM - 1));
    const uint32_t to = lds_addr(lds);
    auto fetch = [&](int stage, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int step = min(stage * Q + q, last);  // (past the end: the last step's bytes, unused)
            const uint32_t at = to + buf * R::STAGE + q * R::STEP;
#pragma unroll
            for (int i = 0; i < R::PER; i++) {
                const uint32_t place = __builtin_amdgcn_readfirstlane(at + 1024 * (wave + R::WAVES * i));
                if (SORTED && 8 * R::WAVES * i >= R::TN) dma16(xp[i] + (int64_t)step * F8_BLOCK, place);
                else dma16_s((8 * R::WAVES * i < R::TN ? w0 : x0) + (int64_t)step * F8_BLOCK, off[i], place);
            }
            if (scales) dma4(xs + step * a.m, __builtin_amdgcn_readfirstlane(at + R::CODES + 256 * wave));
        }
    };
    const int c0 = 16 * ((lane >> 4) ^ (lane & 7)), c1 = 16 * ((4 + (lane >> 4)) ^ (lane & 7));
    const uint8_t *wl = lds + (16 * NF * wn + (lane & 15)) * F8_BLOCK, *xl = lds + (R::TN + 16 * MF * wm + (lane & 15)) * F8_BLOCK;
    const uint8_t *sl = lds + R::CODES + 4 * (16 * MF * wm + (lane & 15));
    const float *sw_of = f8_uniform(ws + (n0 + 16 * NF * wn < a.n ? (n0 + 16 * NF * wn) / F8_BLOCK : 0) * a.blocks);
    f32x4 acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < R::D && s < stages; s++) fetch(s, s);
    int buf = 0, next = R::D;
    const bool strange = f8_any_strange<R::TM, R::TN, R::WAVES>(a, ws, xrow, n0);
    float sw[Q];  // (a step ahead: the scalar loads of a step would be waited for with its reads of LDS)
#pragma unroll
    for (int q = 0; q < Q; q++) sw[q] = f8_scale_at(sw_of + min(q, last));
    for (int stage = 0; stage < stages; stage++) {
        // this wave's part of the stage is in (the stages after it may still be on their way), then every wave's; and
        // every wave has multiplied the stage before, whose place the stage D ahead takes
        if (stage + R::D > stages) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else if (scales) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((R::D - 1) * Q * (R::PER + 1)) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((R::D - 1) * Q * R::PER) : "memory");
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (stage + R::D < stages) fetch(stage + R::D, next);
        next = next + 1 == R::D + 1 ? 0 : next + 1;
        const int o = buf * R::STAGE;
        F8Frag<EXACT> wf[Q][NF];
        float now[Q];
#pragma unroll
        for (int q = 0; q < Q; q++) {
            now[q] = sw[q];
            sw[q] = f8_scale_at(sw_of + min((stage + 1) * Q + q, last));
        }
        if constexpr (EXACT && NF * MF > 4) {  // (the fragments of a step as f16 would take too many registers)
#pragma unroll
            for (int q = 0; q < Q; q++) {
                const int at = o + q * R::STEP;
#pragma unroll
                for (int j = 0; j < NF; j++) wf[0][j].load(wl + at + c0 + 2048 * j, wl + at + c1 + 2048 * j);
#pragma unroll
                for (int i = 0; i < MF; i++) {
                    F8Frag<EXACT> xi;
                    xi.load(xl + at + c0 + 2048 * i, xl + at + c1 + 2048 * i);
                    const float s = Q == 1 || stage * Q + q <= last ? *(const float *)(sl + at + 64 * i) * now[q] : 0.f;
#pragma unroll
                    for (int j = 0; j < NF; j++) {
                        const f32x4 p = F8Frag<EXACT>::product(wf[0][j], xi);
#pragma unroll
                        for (int c = 0; c < 4; c++) acc[i][j][c] = fmaf(p[c], s, acc[i][j][c]);
                    }
                }
            }
        } else {
            F8Frag<EXACT> xf[Q][MF];
            f32x4 p[Q][MF][NF];
            float s[Q][MF];
#pragma unroll
            for (int q = 0; q < Q; q++) {
#pragma unroll
                for (int j = 0; j < NF; j++) wf[q][j].load(wl + o + q * R::STEP + c0 + 2048 * j, wl + o + q * R::STEP + c1 + 2048 * j);
#pragma unroll
                for (int i = 0; i < MF; i++) {
                    xf[q][i].load(xl + o + q * R::STEP + c0 + 2048 * i, xl + o + q * R::STEP + c1 + 2048 * i);
                    s[q][i] = *(const float *)(sl + o + q * R::STEP + 64 * i);
                }
            }
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
                for (int i = 0; i < MF; i++) {
#pragma unroll
                    for (int j = 0; j < NF; j++) p[q][i][j] = F8Frag<EXACT>::product(wf[q][j], xf[q][i]);
                    s[q][i] = Q == 1 || stage * Q + q <= last ? s[q][i] * now[q] : 0.f;  // (past the end the last step again, times nothing)
                }
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
                for (int i = 0; i < MF; i++)
#pragma unroll
                    for (int j = 0; j < NF; j++)
#pragma unroll
                        for (int c = 0; c < 4; c++) acc[i][j][c] = fmaf(p[q][i][j][c], s[q][i], acc[i][j][c]);
        }
        buf = buf + 1 == R::D + 1 ? 0 : buf + 1;
    }
    const bool again = __syncthreads_or(strange);
    f8_finish<T, MF, NF>(a, bias, m0 + 16 * MF * wm, m_end, n0 + 16 * NF * wn, acc, lds + wave * 256 * NF * sizeof(T));
    if (again) f8_strange_tile<T>(a, w, ws, bias, row_at, m0, min(m0 + R::TM, m_end), n0, R::TN);
}

// Many rows of x: tiles of 256 x 256, eight waves of 64 columns x 128 rows, two to a SIMD: one multiplies while the other scales and
// adds. Two LDS stages of 2 x 256 rows x 128 codes and 256 scales, swizzled as in k_f8_tile. A wave's four fragments of W stay in
// registers for the step, x's eight pass by, each read while the one before is multiplied; the next step's first ones while the
// last is, before which all waves meet: the stage of the next step is then in, and this step's, all of which has been read, free for the one after.
// 8,192 x 4,096 x 4,096, bf16: 121 to 142 us by the box (1.9 to 2.3 PFLOP/s), 8,192 cubed 445 to 452 (2.4 to 2.5); matrix pipe 54 % busy, waves at waits and the barrier 29 %,
// waiting to issue 30 %.
template <class T>
__global__ __launch_bounds__(512, 2) void k_f8_big(F8MatArgs a, int tiles_m, int tiles_n) {
    using R = F8Ring<4, 2, 4, 8, 1, 2>;
    using Frag = F8Frag<false>;
    extern __shared__ __align__(1024) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave & 3, wm = wave >> 2, last = a.blocks - 1;
    int64_t m0, n0;
    f8_tile_of_block(tiles_m, tiles_n, R::TM, R::TN, m0, n0);
    const uint8_t *w0 = a.w + n0 * a.rb, *x0 = a.x + m0 * a.rb;
    // load i < 4 of this wave: 8 rows of W from 64 i + 8 wave, then x's likewise
    uint32_t off[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = 64 * (i & 3) + 8 * wave + (lane >> 3);
        off[i] = (uint32_t)min((int64_t)r, (i < 4 ? a.n - n0 : a.m - m0) - 1) * a.rb + 16 * ((lane & 7) ^ (r & 7));
    }
    const float *xs0 = a.xs + m0;
    const uint32_t soff = 4 * (uint32_t)min((int64_t)(64 * wn + lane), a.m - m0 - 1);
    const uint32_t to = lds_addr(lds);
    // load i of a step (8: its scales); past the end the last step's bytes, unused
    auto fetch = [&](int want, int i) __attribute__((always_inline)) {
        const int step = min(want, last);
        const uint32_t stage = to + (want & 1) * R::STAGE;
        if (i < 8) dma16_s((i < 4 ? w0 : x0) + (int64_t)step * F8_BLOCK, off[i], __builtin_amdgcn_readfirstlane(stage + 8192 * i + 1024 * wave));
        else dma4_s((const uint8_t *)(xs0 + step * a.m), soff, __builtin_amdgcn_readfirstlane(stage + R::CODES + 256 * wn));
    };
    const int c0 = 16 * ((lane >> 4) ^ (lane & 7)), c1 = 16 * ((4 + (lane >> 4)) ^ (lane & 7));
    const uint8_t *wl = lds + (64 * wn + (lane & 15)) * F8_BLOCK, *xl = lds + (R::TN + 128 * wm + (lane & 15)) * F8_BLOCK;
    const uint8_t *sl = lds + R::CODES + 4 * (128 * wm + (lane & 15));
    const float *sw_of = f8_uniform(a.ws + (n0 + 64 * wn < a.n ? (n0 + 64 * wn) / F8_BLOCK : 0) * a.blocks);
    f32x4 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    Frag wf[4], xf[2];
    f32x4 p[2][4];  // the sums of these 16 rows, and of those before, which are scaled and added meanwhile
    float sx[2], s = 0.f;
#pragma unroll
    for (int i = 0; i < 9; i++) fetch(0, i);
    const bool strange = f8_any_strange<R::TM, R::TN, R::WAVES>(a, a.ws, [&](int r) { return min(m0 + r, a.m - 1); }, n0);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    fetch(1, 0);
    fetch(1, 1);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        wf[j].load(wl + c0 + 2048 * j, wl + c1 + 2048 * j);
        p[1][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    xf[0].load(xl + c0, xl + c1);
    sx[0] = *(const float *)sl;
    auto add = [&](int i, int j) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 4; c++) acc[i][j][c] = fmaf(p[i & 1][j][c], s, acc[i][j][c]);
    };
    float sw_next = f8_scale_at(sw_of);
    for (int step = 0; step <= last; step++) {
        const float sw = sw_next;
        sw_next = f8_scale_at(sw_of + min(step + 1, last));
        const int o = (step & 1) * R::STAGE, next = R::STAGE - o;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i == 7) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const int at = i < 7 ? o + 2048 * (i + 1) : next;
            xf[(i + 1) & 1].load(xl + at + c0, xl + at + c1);
            sx[(i + 1) & 1] = *(const float *)(sl + (i < 7 ? o + 64 * (i + 1) : next));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                p[i & 1][j] = Frag::product(wf[j], xf[i & 1]);
                __builtin_amdgcn_sched_barrier(0);
                if (i == 7) wf[j].load(wl + next + c0 + 2048 * j, wl + next + c1 + 2048 * j);
                add((i + 7) & 7, j);
                // the next step's loads, two at a time: nine at once after the barrier keep the waves from issuing
                if (j & 1) {
                    const int f = 2 * ((i + 1) & 7) + j / 2;
                    if (f < 9) fetch(i == 7 ? step + 2 : step + 1, f);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            s = sx[i & 1] * sw;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) add(7, j);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // (no load may land in LDS that is another block's)
    const bool again = __syncthreads_or(strange);
    f8_finish<T, 8, 4>(a, a.bias, m0 + 128 * wm, a.m, n0 + 64 * wn, acc, lds + wave * 1024 * sizeof(T));
    if (again) f8_strange_tile<T>(a, a.w, a.ws, a.bias, [](int64_t r) { return r; }, m0, min(m0 + R::TM, a.m), n0, R::TN);
}

// Sorted rows times their experts' matrices: a tile of up to 128 positions, 64 NW columns. 8,192 positions over 128 experts of 2,880 x 2,880: 249 to 256 us, 4.4 TB/s
// (1.1 GB of weights, 47 MB of results); 64 over 256 of 1,024 x 2,048 24 (5.0).
template <class T, int NW, bool EXACT>
__global__ __launch_bounds__(256, 2) void k_f8_experts(F8MatArgs a, int n_blocks) {
    extern __shared__ __align__(1024) uint8_t lds[];
    PileTile tl;
    int nb;
    if (!f8_item_of_block(a.tiles, n_blocks, tl, nb)) return;
    constexpr int COLS = 64 * NW;
    const int lane = threadIdx.x & 63;
    if (tl.expert == a.E) return f8_zeros<T>(a, tl, (int64_t)COLS * nb, COLS);
    const int64_t n0 = (int64_t)COLS * nb + 16 * NW * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n_in = min(n0, a.n - 1);
    F8Operands<1> o;
    o.x = a.x;
    o.xs = a.xs;
    o.m = a.m;
    o.rb = a.rb;
    o.blocks = a.blocks;
    o.w0[0] = a.w + tl.expert * a.w_stride + n_in * a.rb;
    o.ws0[0] = a.ws + tl.expert * a.ws_stride + n_in / F8_BLOCK * a.blocks;
    uint32_t wrow[NW];
#pragma unroll
    for (int j = 0; j < NW; j++) wrow[j] = (uint32_t)min((int64_t)(16 * j + (lane & 15)), a.n - 1 - n_in) * (uint32_t)a.rb + 16 * (lane >> 4);
    f8_by_height(tl.m, [&](auto mb) __attribute__((always_inline)) {
        constexpr int MB = decltype(mb)::value;
        f32x4 acc[MB][NW];
        auto row_at = [&](int64_t pos) __attribute__((always_inline)) { return a.order ? (int64_t)(a.order[pos] / a.K) : pos; };
        const bool odd = f8_stream<MB, NW, 1, EXACT>(lds, o, [&](int r) { return row_at(tl.pos0 + min(r, tl.m - 1)); }, wrow, acc);
        const bool again = __syncthreads_or(odd);
        const float *bias = a.bias ? a.bias + tl.expert * a.n : nullptr;
        f8_finish<T, MB, NW>(a, bias, tl.pos0, tl.pos0 + tl.m, n0, acc, lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 256 * NW * sizeof(T));
        if (again)
            f8_strange_tile<T>(a, a.w + tl.expert * a.w_stride, a.ws + tl.expert * a.ws_stride, bias, row_at, tl.pos0, tl.pos0 + tl.m, (int64_t)COLS * nb, COLS);
    });
}

// dynamic LDS above 64 KB, opted into once per kernel and device
template <class T, int I>
static int f8_allow_lds(const void *kernel, int lds) {
    static std::atomic<bool> set[MAX_DEVICES];
    const int dev = current_device();
    if (set[dev].load(std::memory_order_relaxed)) return CW_OK;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return set_error(CW_EHIP, "f8: %d bytes of LDS", lds);
    set[dev].store(true, std::memory_order_relaxed);
    return CW_OK;
}
template <class T, class R, class Kernel>
static int f8_tiles(const F8MatArgs &a, Kernel kernel, hipStream_t s) {
    const int64_t tm = (a.m + R::TM - 1) / R::TM, tn = (a.n + R::TN - 1) / R::TN;
    if (int rc = f8_allow_lds<T, R::TM>((const void *)kernel, R::LDS)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(R::NT), R::LDS, s, a, (int)tm, (int)tn);
    return check_launch("k_f8_tile");
}
template <class T>
static int f8_matmul(const F8MatArgs &a, int few_groups, int tile_of, hipStream_t s) {
    auto few = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.n + 15) / 16)), dim3(64 * F8_FEW_WAVES), 0, s, a);
        return check_launch("k_f8_few");
    };
    constexpr bool exact = f8_exact_for<T>;
    switch (few_groups) {
    case 0: break;
    case 1: return few(k_f8_few<T, 1, exact>);
    case 2: return few(k_f8_few<T, 2, exact>);
    case 3: return few(k_f8_few<T, 3, exact>);
    case 4: return few(k_f8_few<T, 4, exact>);
    default:
        if constexpr (exact) return few(k_f8_few<T, 5, exact>);
    }
    switch (tile_of) {
    case 0:
        if constexpr (exact) return f8_tiles<T, F8Ring<2, 2, 2, 2, 2, 4>>(a, k_f8_tile<T, exact, false, 2, 2, 2, 2, 2, 4>, s);
        else return f8_tiles<T, F8Ring<4, 2, 1, 2, 4, 2>>(a, k_f8_tile<T, exact, false, 4, 2, 1, 2, 4, 2>, s);
    case 1: return f8_tiles<T, F8Ring<4, 2, 2, 4, 2, 2>>(a, k_f8_tile<T, exact, false, 4, 2, 2, 4, 2, 2>, s);
    default:
        if constexpr (exact) return f8_tiles<T, F8Ring<4, 2, 4, 8, 1, 2>>(a, k_f8_tile<T, exact, false, 4, 2, 4, 8, 1, 2>, s);
        else return f8_tiles<T, F8Ring<4, 2, 4, 8, 1, 2>>(a, k_f8_big<T>, s);
    }
}

template <class T, bool EXACT>
static int f8_experts(const F8MatArgs &a, int64_t tiles, bool sorted, bool four, hipStream_t s) {
    auto go = [&](auto kernel, int cols, int threads, int lds, auto... of) {
        const int blocks = (int)((a.n + cols - 1) / cols);
        hipLaunchKernelGGL(kernel, dim3((unsigned)((tiles * blocks + 7) / 8 * 8)), dim3(threads), lds, s, a, of..., blocks);
        return check_launch("k_f8_experts");
    };
    if (sorted) {
        using R = F8Ring<4, 2, 2, 4, 2, 2>;
        static_assert(R::TM == PILE_TILE, "a tile of positions");
        auto kernel = k_f8_tile<T, EXACT, true, 4, 2, 2, 4, 2, 2>;
        if (int rc = f8_allow_lds<T, 1 + EXACT>((const void *)kernel, R::LDS)) return rc;
        return go(kernel, R::TN, R::NT, R::LDS, 0);
    }
    if (four) return go(k_f8_experts<T, 4, EXACT>, 256, 256, F8Stream<8, 4>::LDS);
    if (int rc = f8_allow_lds<T, 3 + EXACT>((const void *)k_f8_experts<T, 2, EXACT>, F8Stream<8, 2>::LDS)) return rc;
    return go(k_f8_experts<T, 2, EXACT>, 128, 256, F8Stream<8, 2>::LDS);
}

static int check_product(const char *what, int ydtype, int64_t n, int64_t k, int64_t m, int64_t ldy) {
    if (!f8_float_type(ydtype)) return set_error(CW_ENOTSUP, "%s: type %d of y (f32, f16 or bf16)", what, ydtype);
    CW_REQUIRE(n > 0 && k > 0 && m >= 0 && n < (1ll << 31) && m < (1ll << 31), "%s: %lld x %lld, %lld rows of x", what, (long long)n, (long long)k,
               (long long)m);
    if (k > CW_F8_MAX_K) return set_error(CW_ENOTSUP, "%s: rows of %lld above %d", what, (long long)k, CW_F8_MAX_K);
    if (n > 1 << 26) return set_error(CW_ENOTSUP, "%s: %lld rows of w above %d", what, (long long)n, 1 << 26);
    CW_REQUIRE(ldy >= n, "%s: rows of y of %lld %lld apart", what, (long long)n, (long long)ldy);
    return CW_OK;
}
static F8MatArgs product_args(const uint8_t *w, const float *w_scale, int64_t n, int64_t k, const uint8_t *x, const float *x_scale, int64_t m,
                              const float *bias, void *y, int64_t ldy) {
    F8MatArgs a = {};
    a.w = w;
    a.x = x;
    a.ws = w_scale;
    a.xs = x_scale;
    a.bias = bias;
    a.n = n;
    a.m = m;
    a.rb = (int)f8_row_bytes(k);
    a.blocks = (int)f8_blocks(k);
    a.y = y;
    a.ldy = ldy;
    return a;
}

int f8_matmul_experts(const uint8_t *w, int64_t w_stride, const float *w_scale, int n_experts, int64_t n, int64_t k, const uint8_t *x,
                         const float *x_scale, int64_t m, const int32_t *order, int K, int64_t picks, const void *tiles, const float *bias,
                         int ydtype, void *y, int64_t ldy, bool exact, hipStream_t s) {
    if (int rc = check_product("f8_matmul_experts", ydtype, n, k, m, ldy)) return rc;
    CW_REQUIRE(n_experts > 0 && n_experts <= PILE_MAX_EXPERTS, "f8_matmul_experts: %d experts (1..%d supported)", n_experts, PILE_MAX_EXPERTS);
    CW_REQUIRE(K > 0 && picks >= 0 && picks < 1 << 28, "f8_matmul_experts: %lld picks, %d a token", (long long)picks, K);
    CW_REQUIRE(order ? m * K == picks : m == picks, "f8_matmul_experts: %lld rows of x for %lld picks, %d a token", (long long)m, (long long)picks, K);
    CW_REQUIRE(w_stride >= n * f8_row_bytes(k) && w_stride % 16 == 0, "f8_matmul_experts: %lld bytes from an expert's matrix to the next",
               (long long)w_stride);
    const int64_t most = pile_max_tiles(picks, n_experts);
    if (most * ((n + 127) / 128) >= 1 << 23) return set_error(CW_ENOTSUP, "f8_matmul_experts: %lld picks of %lld outputs", (long long)picks, (long long)n);
    if (picks == 0) return CW_OK;
    CW_REQUIRE(w && w_scale && x && x_scale && tiles && y, "f8_matmul_experts: null pointer");
    CW_REQUIRE(f8_aligned(w, 16) && f8_aligned(x, 16) && f8_aligned(tiles, 16), "f8_matmul_experts: codes and tiles must be 16-byte aligned");
    F8MatArgs a = product_args(w, w_scale, n, k, x, x_scale, m, bias, y, ldy);
    a.w_stride = w_stride;
    a.ws_stride = f8_blocks(n) * f8_blocks(k);
    a.tiles = tiles;
    a.order = order;
    a.K = K;
    a.E = n_experts;
    const int cus = (int)resident_blocks(1);
    const bool sorted = most * ((n + 127) / 128) < F8_MAX_TILES && f8_sorted_tiles(exact, n_experts, picks, n, cus);
    const bool four = f8_four_groups(n_experts, picks, n, k, cus);
    if (ydtype == CW_F16) return f8_experts<_Float16, true>(a, most, sorted, four, s);
    if (ydtype == CW_BF16) return f8_experts<bf16_t, false>(a, most, sorted, four, s);
    return exact ? f8_experts<float, true>(a, most, sorted, four, s) : f8_experts<float, false>(a, most, sorted, four, s);
}

}  // namespace cw

using namespace cw;

extern "C" {

int cw_f8_matmul(const uint8_t *w, const float *w_scale, int64_t n, int64_t k, const uint8_t *x, const float *x_scale, int64_t m,
                 const float *bias, int ydtype, void *y, int64_t ldy, cw_stream_t stream) {
    if (int rc = check_product("f8_matmul", ydtype, n, k, m, ldy)) return rc;
    if (m == 0) return CW_OK;
    const int rb = (int)f8_row_bytes(k), cus = (int)resident_blocks(1);
    const bool exact = ydtype != CW_BF16;
    const int few_groups = f8_few_groups(exact, m, n, cus), tile = few_groups ? 0 : f8_pick_tile(exact, m, n, rb, cus);
    if (tile < 0) return set_error(CW_ENOTSUP, "f8_matmul: %lld x %lld outputs", (long long)m, (long long)n);
    CW_REQUIRE(w && w_scale && x && x_scale && y, "f8_matmul: null pointer");
    CW_REQUIRE(f8_aligned(w, 16) && f8_aligned(x, 16), "f8_matmul: codes must be 16-byte aligned");
    const F8MatArgs a = product_args(w, w_scale, n, k, x, x_scale, m, bias, y, ldy);
    hipStream_t s = (hipStream_t)stream;
    if (ydtype == CW_F16) return f8_matmul<_Float16>(a, few_groups, tile, s);
    if (ydtype == CW_BF16) return f8_matmul<bf16_t>(a, few_groups, tile, s);
    return f8_matmul<float>(a, few_groups, tile, s);
}

int cw_f8_matmul_experts(const uint8_t *w, int64_t w_stride, const float *w_scale, int n_experts, int64_t n, int64_t k, const uint8_t *x,
                         const float *x_scale, int64_t m, const int32_t *order, int K, int64_t picks, const void *tiles, const float *bias,
                         int ydtype, void *y, int64_t ldy, cw_stream_t stream) {
    return f8_matmul_experts(w, w_stride, w_scale, n_experts, n, k, x, x_scale, m, order, K, picks, tiles, bias, ydtype, y, ldy, ydtype != CW_BF16,
                             (hipStream_t)stream);
}

}  // extern "C"
