// The product of rows of e4m3 codes on the matrix cores, with scales of 128 columns of k.
#pragma once
#include "cw_f8.h"
#include "cw_f8_dev.h"
#include "cw_gmm_dev.h"
#include "cw_piles.h"

namespace cw {

typedef int i32x8v __attribute__((ext_vector_type(8)));

// A lane's 32 codes of a row of the step, and the product of two rows' on the matrix cores: lane l gives the codes of weight row
// l % 16 (A) and of activation row l % 16 (B), any 32 of the 128 of the step that both operands share (here the 16 from 16 (l / 16)
// and the 16 from 64 + 16 (l / 16)), and gets weight rows 4 (l / 16) + 0..3 of activation row l % 16: four neighbouring outputs
// of one row. The sum of the step alone: what it is multiplied with, the scales of these 128 columns, changes with the step.
//
// v_mfma_f32_16x16x128_f8f6f4 takes the codes as they are. Of the products of 8 neighbouring codes it keeps what is at least 2^(e - 13), e the
// largest sum of two codes' exponents among them, and cuts the rest off towards zero (measured on this part: beside 2^16 a product of 2^3 is kept,
// 2^2 lost, 27.5 becomes 24, whichever of the 8 it is); those sums it adds in f32. So 7 of 8 products lose up to 2^-13 of the largest:
// 7 * 2^-13 of the terms' magnitudes at most, below a quarter of bf16's half step (f16's it may pass); 1.5e-5 of a result of random codes. EXACT: as
// f16, which holds every e4m3 value, at half the rate: each product exact and added in f32 (of 128 widely
// spread products 3e-7 of their magnitudes at the most seen, of random ones 1e-8 of the result), for results in f32 and f16 and for hidden values whose codes hang on them.
template <bool EXACT>
struct F8Frag;
template <>
struct F8Frag<false> {
    i32x8v q;
    __device__ __forceinline__ void load(const uint8_t *a, const uint8_t *b) {
        q = __builtin_shufflevector(*(const i32x4 *)a, *(const i32x4 *)b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ f32x4 product(const F8Frag &w, const F8Frag &x) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.q, x.q, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
    }
};
template <>
struct F8Frag<true> {
    f16x8 h[4];
    __device__ __forceinline__ void load(const uint8_t *a, const uint8_t *b) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint2 v = *(const uint2 *)((i < 2 ? a : b) + 8 * (i & 1));
            const f16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v.x, 1.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v.x, 1.0f, true),
                                __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v.y, 1.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v.y, 1.0f, true)};
            memcpy(&h[i], p, sizeof p);
        }
    }
    static __device__ __forceinline__ f32x4 product(const F8Frag &w, const F8Frag &x) {
        f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; i++) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.h[i], x.h[i], p, 0, 0, 0);
        return p;
    }
};

// A step's sum, below 2^25, is multiplied with the product of two scales in f32, fma(p, sx sw, acc), where both are usual ones: zero, from
// 2^-63 to 2^47, infinite or NaN. Their product is then zero, a normal number, infinite or NaN, and 256 steps' sums of finite ones stay below
// 2^127, in any order. Others, which a program's own codes may have, take their outputs through f8_strange_sums: in 64 bits, so that nothing but
// the result leaves f32's range.
__device__ __forceinline__ bool f8_strange(float s) {
    constexpr uint32_t LOW = 64u << 23, HIGH = 174u << 23, INF = 255u << 23;
    const uint32_t u = __float_as_uint(s) & 0x7FFFFFFFu;
    return u - 1 < LOW - 1 || u - (HIGH + 1) < INF - (HIGH + 1);
}
// Four neighbouring outputs, weight rows w .. w + 3 rb (of `valid`; the last again past them) times one row of x, into acc if one of its scales or
// of theirs is strange (or it is said so): whether is a matter of this row and these weights alone, whatever lies beside them. Slow: a lane reads
// its rows by itself.
__device__ __forceinline__ bool f8_strange_sums(const uint8_t *x, const float *xs, int64_t m, const uint8_t *w, const float *ws, int rb, int valid, f32x4 &acc,
                                                bool strange = false) {
    double sum[4] = {};
#pragma unroll 1
    for (int b = 0; b < rb / F8_BLOCK; b++) {
        const float sx = xs[b * m], sw = ws[b];
        strange |= f8_strange(sx) | f8_strange(sw);
        float p[4] = {};
#pragma unroll 1
        for (int o = b * F8_BLOCK; o < (b + 1) * F8_BLOCK; o += 4) {
            float xv[4], wv[4];
            f8_values4(*(const uint32_t *)(x + o), xv);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f8_values4(*(const uint32_t *)(w + (int64_t)min(i, valid - 1) * rb + o), wv);
#pragma unroll
                for (int c = 0; c < 4; c++) p[i] = fmaf(xv[c], wv[c], p[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) sum[i] = fma((double)p[i], (double)sx * sw, sum[i]);
    }
    if (strange)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = (float)sum[i];
    return strange;
}

// A weights' scale by a scalar load, at a wave-uniform place. (A vector load, which the compiler makes of it beside the inline waits, returns after
// all loads asked for before it: with the weights of the steps ahead in flight it waits for them.)
template <class P>
__device__ __forceinline__ const P *f8_uniform(const P *p) {
    const uint64_t u = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
    return (const P *)(lo | (uint64_t)hi << 32);
}
__device__ __forceinline__ float f8_scale_at(const float *p) { return *(const __attribute__((address_space(4))) float *)(uint64_t)p; }

// Results in f32 and f16 have exact products; bf16's rounding covers what the 8-bit instruction leaves out.
template <class T>
constexpr bool f8_exact_for = !std::is_same_v<T, bf16_t>;

// A block of four waves over a stream of weights: MB blocks of 16 activation rows shared by all of them, NW groups of 16 weight rows for
// each wave (of MATS matrices, NW / MATS of each), k in steps of 512 / NW codes (NW 2: 256, where the weights' bytes bound; NW 4: 128,
// half the reads of LDS for a product, where many rows share the weights). A wave's weights, which no other wave reads, come
// straight into its registers, a whole step ahead: the step's neighbouring bytes of a row asked for together. The activations
// and their scales go through registers (two steps ahead) into two LDS stages, one barrier a step; chunk c (16 bytes) of row r lies at
// chunk c ^ (r % chunks of a row) of its LDS row: the reads of one chunk touch all banks once.
template <int MB, int NW>
struct F8Stream {
    static constexpr int WIDE = 512 / NW, CHUNKS = WIDE / 16, Q = WIDE / F8_BLOCK, CODES = 16 * MB * WIDE, STAGE = CODES + 16 * MB * Q * 4, LDS = 2 * STAGE;
    static constexpr int ROWS = 64 / CHUNKS, LOADS = 16 * MB / ROWS, PER = (LOADS + 3) / 4;  // rows of a load, loads of a stage and of a wave
    static_assert(16 * MB * Q <= 256, "a scale a thread");
};
// What a block multiplies: xrow(r): x's row of row r < 16 MB of the tile (any valid row past its end), of rb codes with `blocks` scales
// m apart; w0[i]: the matrices' first rows of this wave (wave-uniform), ws0[i]: their scales; wrow[j]: the lane's offset of its weight row of group
// j, + 16 (lane / 16). True if the thread saw a strange scale.
template <int MATS>
struct F8Operands {
    const uint8_t *x, *w0[MATS];
    const float *xs, *ws0[MATS];
    int64_t m;
    int rb, blocks;
};
template <int MB, int NW, int MATS, bool EXACT, class XRow>
__device__ __forceinline__ bool f8_stream(uint8_t *lds, const F8Operands<MATS> &a, XRow xrow, const uint32_t (&wrow)[NW], f32x4 (&acc)[MB][NW]) {
    using S = F8Stream<MB, NW>;
    constexpr int WIDE = S::WIDE, Q = S::Q;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = (a.rb + WIDE - 1) / WIDE, chunk = lane % S::CHUNKS;
    // load i of this wave: the rows from ROWS (wave + 4 i) (with fewer loads than waves, some twice: the same bytes to
    // the same place)
    const uint8_t *xp[S::PER];
    int xl[S::PER];
#pragma unroll
    for (int i = 0; i < S::PER; i++) {
        const int r = S::ROWS * ((wave + 4 * i) % S::LOADS) + lane / S::CHUNKS;
        xp[i] = a.x + xrow(r) * (int64_t)a.rb;
        xl[i] = r * WIDE + 16 * (chunk ^ (r % S::CHUNKS));
    }
    // this thread's scale of a step (with fewer scales than threads, some twice): that of row at % 16 MB, block at / 16 MB
    const int st = threadIdx.x % (16 * MB * Q), sb = st / (16 * MB);
    const float *sp = a.xs + xrow(st % (16 * MB));
    i32x4 xr[S::PER], w[2][NW][2 * Q];
    const float *ws[MATS];
    float xsr = 0.f, sw[MATS][Q];
#pragma unroll
    for (int i = 0; i < MATS; i++) ws[i] = f8_uniform(a.ws0[i]);
    auto fetch_sw = [&](int step) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MATS; i++)
#pragma unroll
            for (int q = 0; q < Q; q++) sw[i][q] = f8_scale_at(ws[i] + min(step * Q + q, a.blocks - 1));
    };
    bool odd = false;
    // the lane's chunk of k of a step, and whether the row has it (past its end: its last line, not used)
    auto fetch_x = [&](int step) __attribute__((always_inline)) {
        const int o = min(step * WIDE + 16 * chunk, a.rb - 16);
#pragma unroll
        for (int i = 0; i < S::PER; i++) xr[i] = *(const i32x4 *)(xp[i] + o);
        xsr = sp[min(step * Q + sb, a.blocks - 1) * a.m];
    };
    auto store_x = [&](int step) __attribute__((always_inline)) {
        const bool in = step * WIDE + 16 * chunk < a.rb;
        uint8_t *to = lds + (step & 1) * S::STAGE;
#pragma unroll
        for (int i = 0; i < S::PER; i++) *(i32x4 *)(to + xl[i]) = in ? xr[i] : i32x4{0, 0, 0, 0};
        ((float *)(to + S::CODES))[st] = step * Q + sb < a.blocks ? xsr : 0.f;
        odd |= f8_strange(xsr);
    };
    auto fetch_w = [&](int step, i32x4 (&v)[NW][2 * Q]) __attribute__((always_inline)) {
        const int o = min(step * WIDE, a.rb - 128), o2 = min(step * WIDE + 128, a.rb - 128);
#pragma unroll
        for (int j = 0; j < NW; j++) {
            const uint8_t *b = a.w0[j / (NW / MATS)];
            v[j][0] = *(const i32x4 *)(b + o + wrow[j]);
            v[j][1] = *(const i32x4 *)(b + o + 64 + wrow[j]);
            if constexpr (Q == 2) {
                v[j][2] = *(const i32x4 *)(b + o2 + wrow[j]);
                v[j][3] = *(const i32x4 *)(b + o2 + 64 + wrow[j]);
            }
        }
    };
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int j = 0; j < NW; j++) acc[mb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto body = [&](int step, i32x4 (&now)[NW][2 * Q], i32x4 (&next)[NW][2 * Q]) __attribute__((always_inline)) {
        // every wave's part of the stage is in LDS, and every wave has multiplied the stage before it, whose buffer
        // the next one takes
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        store_x(step + 1);
        __builtin_amdgcn_sched_barrier(0);
        fetch_x(step + 2);
        fetch_w(step + 1, next);
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t *b = lds + (step & 1) * S::STAGE + (lane & 15) * WIDE;
        const float *sx = (const float *)(lds + (step & 1) * S::STAGE + S::CODES) + (lane & 15);
        float sn[MATS][Q];  // (the next step's are asked for a step ahead)
#pragma unroll
        for (int i = 0; i < MATS; i++)
#pragma unroll
            for (int q = 0; q < Q; q++) {
                odd |= f8_strange(sw[i][q]);
                sn[i][q] = step * Q + q < a.blocks ? sw[i][q] : 0.f;  // (past the end the last one again, which may be infinite)
            }
        fetch_sw(step + 1);
#pragma unroll
        for (int q = 0; q < Q; q++) {
            auto frag = [&](int mb) __attribute__((always_inline)) {
                F8Frag<EXACT> f;
                const uint8_t *p = b + mb * 16 * WIDE;
                f.load(p + 16 * ((8 * q + (lane >> 4)) ^ (lane & (S::CHUNKS - 1))), p + 16 * ((8 * q + 4 + (lane >> 4)) ^ (lane & (S::CHUNKS - 1))));
                return f;
            };
            auto add = [&](int mb, int j, f32x4 p) __attribute__((always_inline)) {
                const float s = sx[q * 16 * MB + 16 * mb] * sn[j / (NW / MATS)][q];
#pragma unroll
                for (int c = 0; c < 4; c++) acc[mb][j][c] = fmaf(p[c], s, acc[mb][j][c]);
                asm volatile("" : "+v"(acc[mb][j]));  // (here and now: sunk to the next step, the products would need registers of their own)
            };
            if constexpr (EXACT) {
                // a weight's halves are made once, a row's for each group of weights: of both there is no room for all
#pragma unroll
                for (int j = 0; j < NW; j++) {
                    F8Frag<true> wf;
                    wf.load((const uint8_t *)&now[j][2 * q], (const uint8_t *)&now[j][2 * q + 1]);
#pragma unroll
                    for (int mb = 0; mb < MB; mb++) {
                        add(mb, j, F8Frag<true>::product(wf, frag(mb)));
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            } else {
                F8Frag<false> x = frag(0), wf[NW];
#pragma unroll
                for (int j = 0; j < NW; j++) wf[j].load((const uint8_t *)&now[j][2 * q], (const uint8_t *)&now[j][2 * q + 1]);
#pragma unroll
                for (int mb = 0; mb < MB; mb++) {
                    // the next fragment of x is read while this one is multiplied (the fences keep the compiler from reading
                    // them all at once)
                    F8Frag<false> xn = x;
                    if (mb + 1 < MB) xn = frag(mb + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    f32x4 p[NW];
#pragma unroll
                    for (int j = 0; j < NW; j++) p[j] = F8Frag<false>::product(wf[j], x);
#pragma unroll
                    for (int j = 0; j < NW; j++) add(mb, j, p[j]);
                    __builtin_amdgcn_sched_barrier(0);
                    x = xn;
                }
            }
        }
    };
    fetch_sw(0);
    fetch_x(0);
    store_x(0);
    fetch_x(1);
    __builtin_amdgcn_sched_barrier(0);
    fetch_w(0, w[0]);
    for (int step = 0; step < steps; step += 2) {  // (a step past the end multiplies zeros)
        body(step, w[0], w[1]);
        body(step + 1, w[1], w[0]);
    }
    return odd;
}
// The item of a block: blocks go to the eight dies in turn; each die takes a contiguous range of the items, an expert's
// blocks of W one after the other and its tiles side by side for each, so that an expert's rows and weights are read by
// one die and not by all, the weights once for all its tiles.
__device__ __forceinline__ bool f8_item_of_block(const void *list, int n_blocks, PileTile &tl, int &nb) {
    const PileTile *tiles = pile_tiles(list);
    const int64_t total = (int64_t)*(const int *)list * n_blocks, per = total >> 3;
    const int die = blockIdx.x & 7, at = blockIdx.x >> 3, rest = (int)(total & 7);
    if (at >= per + (die < rest)) return false;
    const int64_t item = die * per + min(die, rest) + at;
    const PileTile any = tiles[__builtin_amdgcn_readfirstlane((int)(item / n_blocks))];  // a tile of the item's expert
    const int in = (int)(item - (int64_t)any.first * n_blocks);
    nb = __builtin_amdgcn_readfirstlane(in / any.of);
    if (any.of == 1) tl = any;
    else tl = tiles[__builtin_amdgcn_readfirstlane(any.first + in - nb * any.of)];
    tl.expert = __builtin_amdgcn_readfirstlane(tl.expert);
    tl.pos0 = __builtin_amdgcn_readfirstlane(tl.pos0);
    tl.m = __builtin_amdgcn_readfirstlane(tl.m);
    return true;
}
// f(the number of 16s that a tile's positions take), of those that a kernel is built for
template <class F>
__device__ __forceinline__ void f8_by_height(int m, F f) {
    if (m <= 16) f(std::integral_constant<int, 1>{});
    else if (m <= 32) f(std::integral_constant<int, 2>{});
    else if (m <= 48) f(std::integral_constant<int, 3>{});
    else if (m <= 64) f(std::integral_constant<int, 4>{});
    else if (m <= 80) f(std::integral_constant<int, 5>{});
    else if (m <= 96) f(std::integral_constant<int, 6>{});
    else f(std::integral_constant<int, 8>{});
}

// four neighbouring outputs
template <class T>
__device__ __forceinline__ void f8_store4(T *y, int valid, f32x4 v, const float (&b)[4]) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = v[i] + b[i];
    store_row<4>(y, valid, f);
}

}  // namespace cw
