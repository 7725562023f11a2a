// Products of 8-bit integer rows with 8-bit integer matrices (gfx950).
#include <atomic>

#include "cw_i8.h"
#include "cw_i8_rules.h"
#include "cw_i8_tile.h"
#include "cw_mfma.h"

namespace cw {

struct I8MatArgs {
    const uint8_t *w, *x;
    const float *ws, *xs, *bias;
    int64_t n, m;
    int rb;      // bytes of a row
    void *y;
    int64_t ldy;
};

// The formula of an output, the same in every kernel, so that a row's results do not depend on the rows beside it, whose number
// picks the kernel: in f32, fma(sum, sx sw, bias), where both scales are usual ones, zero or from 2^-63 to 2^63 (their product is
// zero or a normal number), else in 64 bits. (For all in 64 bits 8,192 rows of 4096 x 4096 took 135 us in a graph instead of 126.)
struct ScaleRange {
    uint32_t least = ~0u, most = 0;
    __device__ __forceinline__ void add(float s) {
        const uint32_t u = __float_as_uint(s) & 0x7FFFFFFFu;
        least = min(least, u - 1);  // (zero: the largest)
        most = max(most, u);
    }
    __device__ __forceinline__ bool usual() const { return least >= (64u << 23) - 1 && most <= 190u << 23; }
};
// four outputs of row m from column n. USUAL: all their scales are
template <class T, bool USUAL>
__device__ __forceinline__ void i8_store4(const I8MatArgs &a, int64_t m, int64_t n, i32x4 v, float sx, const float (&sw)[4], const float (&b)[4]) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[i] = fmaf((float)v[i], sx * sw[i], b[i]);
        if constexpr (!USUAL) {
            ScaleRange r;
            r.add(sx);
            r.add(sw[i]);
            if (!r.usual()) f[i] = scaled(v[i], (double)sx * sw[i], b[i]);
        }
        asm("" : "+v"(f[i]));  // (in f32: some kernels would fuse the fma with f16's conversion, others not)
    }
    store_row<4>((T *)a.y + m * a.ldy + n, a.n - n < 4 ? (int)(a.n - n) : 4, f);
}

// A wave's sums scaled and stored: rows of x from m0, of W from n0. All scales are loaded first, from clamped
// places: loads inside the bounds checks would be waited for one after the other (32 us a tile of 256 x 256).
template <class T, int MB, int NW>
__device__ __forceinline__ void i8_finish(const I8MatArgs &a, int64_t m0, int64_t n0, const i32x4 (&acc)[MB][NW]) {
    const int lane = threadIdx.x & 63;
    const int64_t m = m0 + (lane & 15), n = n0 + 4 * (lane >> 4);
    float sx[MB], sw[NW][4], b[NW][4];
#pragma unroll
    for (int i = 0; i < MB; i++) sx[i] = a.xs[min(m + 16 * i, a.m - 1)];
    if (n0 + 16 * NW <= a.n) {  // (whole for the wave: four neighbours at a time)
#pragma unroll
        for (int j = 0; j < NW; j++) memcpy(sw[j], a.ws + n + 16 * j, 16);
        if (a.bias)
#pragma unroll
            for (int j = 0; j < NW; j++) memcpy(b[j], a.bias + n + 16 * j, 16);
    } else {
#pragma unroll
        for (int j = 0; j < NW; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int64_t at = min(n + 16 * j + c, a.n - 1);
                sw[j][c] = a.ws[at];
                b[j][c] = a.bias ? a.bias[at] : 0.f;
            }
    }
    if (!a.bias)
#pragma unroll
        for (int j = 0; j < NW; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) b[j][c] = 0.f;
    auto store = [&](auto usual) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MB; i++) {
            if (m + 16 * i >= a.m) continue;
#pragma unroll
            for (int j = 0; j < NW; j++)
                if (n + 16 * j < a.n) i8_store4<T, usual.value>(a, m + 16 * i, n + 16 * j, acc[i][j], sx[i], sw[j], b[j]);
        }
    };
    ScaleRange r;
#pragma unroll
    for (int i = 0; i < MB; i++) r.add(sx[i]);
#pragma unroll
    for (int j = 0; j < NW; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) r.add(sw[j][c]);
    if (__all(r.usual())) store(std::true_type{});
    else store(std::false_type{});
}

// Blocks go to the eight dies in turn: each die gets a contiguous range of tiles, in panels of four tiles of W, so that
// those which it runs at once share both operands through its cache (4096 x 4096 at 512 rows in tiles of 64 x 128:
// 23.7 us with the tiles in block order, each die reading all of W).
__device__ __forceinline__ void i8_tile_of_block(int tiles_m, int tiles_n, int tm, int tn, int64_t &m0, int64_t &n0) {
    const int total = tiles_m * tiles_n, die = blockIdx.x & 7, per = total >> 3, rest = total & 7;
    const int id = die * per + min(die, rest) + (int)(blockIdx.x >> 3);
    const int panel = id / (4 * tiles_m), width = min(4, tiles_n - 4 * panel), in = id - panel * 4 * tiles_m;
    m0 = (int64_t)__builtin_amdgcn_readfirstlane(in / width) * tm;
    n0 = (int64_t)__builtin_amdgcn_readfirstlane(4 * panel + in % width) * tn;
}

// Many rows of x: tiles of 256 x 256, four waves of 128 x 128 each (one to a SIMD: its sums take half the
// registers). Both operands go through two LDS stages of 2 x 256 rows x 128 codes by direct global-to-LDS loads
// of whole cache lines, swizzled as in i8_loop. A half step's 16 fragments are read from LDS while the half before
// it is multiplied: those of step s, half 1 during half 0; those of step s + 1, half 0 during half 1, before
// which all waves meet: the stage of s + 1 is then in (its loads were issued a step before), and that of s, all
// whose fragments are in registers, is free for s + 2.
constexpr int I8_BIG = 256, I8_BIG_STAGE = 2 * I8_BIG * I8_STEP;
template <class T>
__global__ __launch_bounds__(256, 1) void k_i8_big(I8MatArgs a, int tiles_m, int tiles_n) {
    extern __shared__ __align__(1024) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), steps = a.rb / I8_STEP;
    int64_t m0, n0;
    i8_tile_of_block(tiles_m, tiles_n, I8_BIG, I8_BIG, m0, n0);
    const uint8_t *w0 = a.w + n0 * a.rb, *x0 = a.x + m0 * a.rb;
    const int wn = wave & 1, wm = wave >> 1;
    uint32_t wo[8], xo[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = 8 * (wave + 4 * i) + (lane >> 3), c = 16 * ((lane & 7) ^ (r & 7));
        wo[i] = (uint32_t)min((int64_t)r, a.n - 1 - n0) * a.rb + c;
        xo[i] = (uint32_t)min((int64_t)r, a.m - 1 - m0) * a.rb + c;
    }
    const uint32_t to = lds_addr(lds) + 1024 * wave;
    const int last = steps - 1;
    auto fetch = [&](int want, int i, bool of_x) __attribute__((always_inline)) {
        const int step = min(want, last);  // (past the end: the last step's bytes, unused)
        const uint32_t at = to + (want & 1) * I8_BIG_STAGE + 4096 * i;
        if (of_x) dma16_s(x0 + (int64_t)step * I8_STEP, xo[i], __builtin_amdgcn_readfirstlane(at + I8_BIG_STAGE / 2));
        else dma16_s(w0 + (int64_t)step * I8_STEP, wo[i], __builtin_amdgcn_readfirstlane(at));
    };
    const uint8_t *wl = lds + (128 * wn + (lane & 15)) * I8_STEP, *xl = lds + I8_BIG_STAGE / 2 + (128 * wm + (lane & 15)) * I8_STEP;
    const int c[2] = {16 * ((lane >> 4) ^ (lane & 7)), 16 * ((4 + (lane >> 4)) ^ (lane & 7))};
    i32x4 w[2][8], x[2][8], acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        fetch(0, i, false);
        fetch(0, i, true);
    }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; i++) {
        fetch(1, i, false);
        fetch(1, i, true);
        w[0][i] = *(const i32x4 *)(wl + c[0] + 2048 * i);
        x[0][i] = *(const i32x4 *)(xl + c[0] + 2048 * i);
    }
    for (int step = 0; step < steps; step++) {
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            if (kk) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const int from = ((step + kk) & 1) * I8_BIG_STAGE;  // (after the last step: a stage that is not used)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // spread between the products: two fragments' reads of the next half (W's first, all of which its first
                // products take) and two loads of the stage after next
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const int f = 2 * i + q;
                    if (f < 8) w[kk ^ 1][f] = *(const i32x4 *)(wl + from + c[kk ^ 1] + 2048 * f);
                    else x[kk ^ 1][f - 8] = *(const i32x4 *)(xl + from + c[kk ^ 1] + 2048 * (f - 8));
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 4 * q; j < 4 * q + 2; j++) acc[i][j] = mfma_i8(w[kk][j], x[kk][i], acc[i][j]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (kk) fetch(step + 2, i, q);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 4 * q + 2; j < 4 * q + 4; j++) acc[i][j] = mfma_i8(w[kk][j], x[kk][i], acc[i][j]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (no load may land in LDS that is another block's)
    i8_finish<T, 8, 8>(a, m0 + 128 * wm, n0 + 128 * wn, acc);
}

// Fewer rows than fill the device with such tiles: tiles of 32 FM x 32 FN, eight waves: two groups of four (16 FM x
// 16 FN each), one for each half of a step. A ring of LDS stages keeps 96 to 128 KB of loads in flight on a CU, for which
// these tiles wait (51 % of the waves' cycles at 77 rows of 4001 x 2880); the groups' integer sums meet in LDS.
template <int FM, int FN>
struct I8Ring {
    static constexpr int TM = 32 * FM, TN = 32 * FN, STAGE = (TM + TN) * I8_STEP, STAGES = 163840 / STAGE < 8 ? 163840 / STAGE : 8;
    static constexpr int PER = STAGE / 8192, LDS = STAGES * STAGE;  // loads of a wave
    static_assert(LDS >= 4 * 64 * 16 * FM * FN && LDS <= 160 * 1024, "the sums of a group fit the ring, the ring the CU");
};
template <class T, int FM, int FN>
__global__ __launch_bounds__(512, 2) void k_i8_ring(I8MatArgs a, int tiles_m, int tiles_n) {
    using R = I8Ring<FM, FN>;
    extern __shared__ __align__(1024) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), steps = a.rb / I8_STEP;
    int64_t m0, n0;
    i8_tile_of_block(tiles_m, tiles_n, R::TM, R::TN, m0, n0);
    const int g = wave >> 2, wn = wave & 1, wm = (wave >> 1) & 1;
    // a stage: TN rows of W, then TM of x; load i of this wave: 8 rows from 8 (wave + 8 i)
    uint32_t off[R::PER];
#pragma unroll
    for (int i = 0; i < R::PER; i++) {
        const int r = 8 * (wave + 8 * i) + (lane >> 3);
        const int64_t row = r < R::TN ? min((int64_t)r, a.n - 1 - n0) : min((int64_t)r - R::TN, a.m - 1 - m0);
        off[i] = (uint32_t)row * a.rb + 16 * ((lane & 7) ^ (r & 7));
    }
    const uint8_t *w0 = a.w + n0 * a.rb, *x0 = a.x + m0 * a.rb;
    const uint32_t to = lds_addr(lds) + 1024 * wave;
    auto fetch = [&](int step, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < R::PER; i++)
            dma16_s((8 * (wave + 8 * i) < R::TN ? w0 : x0) + (int64_t)step * I8_STEP, off[i], __builtin_amdgcn_readfirstlane(to + buf * R::STAGE + 8192 * i));
    };
    const int at = 16 * ((4 * g + (lane >> 4)) ^ (lane & 7)) + (lane & 15) * I8_STEP;
    const uint8_t *wl = lds + 16 * FN * wn * I8_STEP + at, *xl = lds + (R::TN + 16 * FM * wm) * I8_STEP + at;
    i32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    constexpr int D = R::STAGES - 1;
    for (int s = 0; s < D && s < steps; s++) fetch(s, s);
    int buf = 0, next = D;
    for (int step = 0; step < steps; step++) {
        // this wave's part of the stage is in (the stages after it may still be on their way), then every wave's; and
        // every wave has multiplied the stage before, whose place the stage D ahead takes
        if (step + D <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((D - 1) * R::PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (step + D < steps) fetch(step + D, next);
        next = next + 1 == R::STAGES ? 0 : next + 1;
        i32x4 w[FN], x[FM];
#pragma unroll
        for (int j = 0; j < FN; j++) w[j] = *(const i32x4 *)(wl + buf * R::STAGE + 2048 * j);
#pragma unroll
        for (int i = 0; i < FM; i++) x[i] = *(const i32x4 *)(xl + buf * R::STAGE + 2048 * i);
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) acc[i][j] = mfma_i8(w[j], x[i], acc[i][j]);
        buf = buf + 1 == R::STAGES ? 0 : buf + 1;
    }
    __syncthreads();
    i32x4 *sum = (i32x4 *)lds + (wave & 3) * FM * FN * 64 + lane;
    if (g) {
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) sum[(i * FN + j) * 64] = acc[i][j];
    }
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] += sum[(i * FN + j) * 64];
    i8_finish<T, FM, FN>(a, m0 + 16 * FM * wm, n0 + 16 * FN * wn, acc);
}

// Few rows of x: a block takes 16 rows of W and up to 16 MB of x over all of k, its waves the steps of 128 codes in
// turn, both operands straight from memory into registers (no byte of either is used by two waves of a block). The
// waves' sums meet in LDS: integers, so in any order the same. One row of 8192 x 8192: 14 us, 4.8 TB/s (16 waves, or
// two to four steps' loads at a time, when it took 15.0: 15.0 to 18.8, fewer blocks fit a CU); 2048 x 2048: 3.8 us, of which the
// launch and one round trip are most.
template <class T, int MB>
__global__ __launch_bounds__(64 * I8_FEW_WAVES) void k_i8_few(I8MatArgs a) {
    __shared__ i32x4 part[I8_FEW_WAVES][MB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = a.rb / I8_STEP, at = 16 * (lane >> 4);
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const uint8_t *w0 = a.w + n0 * a.rb;
    const uint32_t wrow = (uint32_t)(min(lane & 15, (int)(a.n - 1 - n0)) * a.rb + at);
    uint32_t xrow[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) xrow[i] = (uint32_t)(min(16 * i + (lane & 15), (int)a.m - 1) * a.rb + at);
    i32x4 acc[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) acc[i] = i32x4{0, 0, 0, 0};
    for (int step = wave; step < steps; step += I8_FEW_WAVES) {
        i32x4 w[2], x[MB][2];
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            const int64_t o = (int64_t)step * I8_STEP + 64 * kk;
            w[kk] = load16(w0 + o + wrow);
#pragma unroll
            for (int i = 0; i < MB; i++) x[i][kk] = load16(a.x + o + xrow[i]);
        }
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
            for (int i = 0; i < MB; i++) acc[i] = mfma_i8(w[kk], x[i][kk], acc[i]);
    }
    const int64_t m = 16 * (wave % MB) + (lane & 15), n = n0 + 4 * (lane >> 4);
    const float sx = a.xs[min(m, a.m - 1)];
    float sw[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        sw[i] = a.ws[min(n + i, a.n - 1)];
        b[i] = a.bias ? a.bias[min(n + i, a.n - 1)] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < MB; i++) part[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave >= MB || m >= a.m || n >= a.n) return;
    i32x4 v = part[0][wave][lane];
#pragma unroll
    for (int o = 1; o < I8_FEW_WAVES; o++) v += part[o][wave][lane];
    ScaleRange r;
    r.add(sx);
#pragma unroll
    for (int i = 0; i < 4; i++) r.add(sw[i]);
    if (__all(r.usual())) i8_store4<T, true>(a, m, n, v, sx, sw, b);
    else i8_store4<T, false>(a, m, n, v, sx, sw, b);
}

// dynamic LDS above 64 KB, opted into once per kernel and device
template <class T>
static int i8_allow_lds(const void *kernel, int i, int lds) {
    static std::atomic<bool> set[MAX_DEVICES][4];
    const int dev = current_device();
    if (set[dev][i].load(std::memory_order_relaxed)) return CW_OK;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
        return set_error(CW_EHIP, "i8_matmul: %d bytes of LDS", lds);
    set[dev][i].store(true, std::memory_order_relaxed);
    return CW_OK;
}

template <class T>
static int i8_matmul(const I8MatArgs &a, int few_groups, int tile_of, hipStream_t s) {
    auto few = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.n + 15) / 16)), dim3(64 * I8_FEW_WAVES), 0, s, a);
        return check_launch("k_i8_few");
    };
    auto tile = [&](auto kernel, int threads, int lds) {
        const I8TileTime &t = I8_TILES[tile_of];
        const int64_t tm = (a.m + t.tm - 1) / t.tm, tn = (a.n + t.tn - 1) / t.tn;
        if (int rc = i8_allow_lds<T>((const void *)kernel, tile_of, lds)) return rc;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(threads), lds, s, a, (int)tm, (int)tn);
        return check_launch("k_i8_tile");
    };
    if (few_groups) return few_groups == 1 ? few(k_i8_few<T, 1>) : few_groups == 2 ? few(k_i8_few<T, 2>) : few(k_i8_few<T, 4>);
    switch (tile_of) {
    case 0: return tile(k_i8_ring<T, 2, 2>, 512, I8Ring<2, 2>::LDS);
    case 1: return tile(k_i8_ring<T, 2, 4>, 512, I8Ring<2, 4>::LDS);
    case 2: return tile(k_i8_ring<T, 4, 4>, 512, I8Ring<4, 4>::LDS);
    default: return tile(k_i8_big<T>, 256, 2 * I8_BIG_STAGE);
    }
}

}  // namespace cw

using namespace cw;

extern "C" {

int cw_i8_matmul(const int8_t *w, const float *w_scale, int64_t n, int64_t k, const int8_t *x, const float *x_scale, int64_t m,
                 const float *bias, int ydtype, void *y, int64_t ldy, cw_stream_t stream) {
    if (!i8_float_type(ydtype)) return set_error(CW_ENOTSUP, "i8_matmul: type %d of y (f32, f16 or bf16)", ydtype);
    CW_REQUIRE(n > 0 && k > 0 && m >= 0 && n < (1ll << 31) && m < (1ll << 31), "i8_matmul: %lld x %lld, %lld rows of x", (long long)n,
               (long long)k, (long long)m);
    if (k > CW_I8_MAX_K) return set_error(CW_ENOTSUP, "i8_matmul: rows of %lld above %d", (long long)k, CW_I8_MAX_K);
    if (n > 1 << 26) return set_error(CW_ENOTSUP, "i8_matmul: %lld rows of w above %d", (long long)n, 1 << 26);
    CW_REQUIRE(ldy >= n, "i8_matmul: rows of y of %lld %lld apart", (long long)n, (long long)ldy);
    if (m == 0) return CW_OK;
    const int rb = (int)i8_row_bytes(k), few_groups = i8_few_groups(m, n, rb), tile = few_groups ? 0 : i8_pick_tile(m, n, rb, (int)resident_blocks(1));
    if (tile < 0) return set_error(CW_ENOTSUP, "i8_matmul: %lld x %lld outputs", (long long)m, (long long)n);
    CW_REQUIRE(w && w_scale && x && x_scale && y, "i8_matmul: null pointer");
    CW_REQUIRE(i8_aligned(w, 16) && i8_aligned(x, 16), "i8_matmul: codes must be 16-byte aligned");
    I8MatArgs a = {};
    a.w = (const uint8_t *)w;
    a.x = (const uint8_t *)x;
    a.ws = w_scale;
    a.xs = x_scale;
    a.bias = bias;
    a.n = n;
    a.m = m;
    a.rb = rb;
    a.y = y;
    a.ldy = ldy;
    hipStream_t s = (hipStream_t)stream;
    if (ydtype == CW_F16) return i8_matmul<_Float16>(a, few_groups, tile, s);
    if (ydtype == CW_BF16) return i8_matmul<bf16_t>(a, few_groups, tile, s);
    return i8_matmul<float>(a, few_groups, tile, s);
}

}  // extern "C"
