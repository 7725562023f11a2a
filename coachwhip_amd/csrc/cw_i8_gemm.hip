// Products of 8-bit integer rows with 8-bit integer matrices (gfx950).
#include "cw_i8.h"
#include "cw_i8_tile.h"

namespace cw {

struct I8MatArgs {
    const uint8_t *w, *x;
    const float *ws, *xs, *bias;
    int64_t n, m;
    int rb;      // bytes of a row
    void *y;
    int64_t ldy;
};

// four outputs of row m from column n, scaled: sum * (sx sw) + bias
template <class T>
__device__ __forceinline__ void i8_store4(const I8MatArgs &a, int64_t m, int64_t n, i32x4 v, float sx, const float (&sw)[4], const float (&b)[4]) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = fmaf((float)v[i], sx * sw[i], b[i]);
    store_row<4>((T *)a.y + m * a.ldy + n, a.n - n < 4 ? (int)(a.n - n) : 4, f);
}

// Tiles of 128 rows of x and 256 rows of W: four waves of 64 weight rows each.
template <class T, int MB, int NW>
__global__ __launch_bounds__(256, 2) void k_i8_tile(I8MatArgs a, int tiles_m) {
    extern __shared__ __align__(1024) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t m0 = (int64_t)(blockIdx.x % tiles_m) * 16 * MB, n0 = (int64_t)(blockIdx.x / tiles_m) * 64 * NW + wave * 16 * NW;
    const int64_t nb = min(n0, a.n - 1);
    uint32_t wrow[NW];
#pragma unroll
    for (int j = 0; j < NW; j++) wrow[j] = (uint32_t)((min(n0 + 16 * j + (lane & 15), a.n - 1) - nb) * a.rb + 16 * (lane >> 4));
    i32x4 acc[MB][NW];
    const uint8_t *w0[1] = {a.w + nb * a.rb};
    i8_loop<MB, NW, 4, 1>(lds, a.x + m0 * a.rb, [&](int r) { return (uint32_t)((min(m0 + r, a.m - 1) - m0) * a.rb); }, w0, wrow,
                       a.rb / I8_STEP, acc);
    float sw[NW][4], b[NW][4];
#pragma unroll
    for (int j = 0; j < NW; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t n = min(n0 + 16 * j + 4 * (lane >> 4) + i, a.n - 1);
            sw[j][i] = a.ws[n];
            b[j][i] = a.bias ? a.bias[n] : 0.f;
        }
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        const int64_t m = m0 + 16 * mb + (lane & 15);
        if (m >= a.m) continue;
        const float sx = a.xs[m];
#pragma unroll
        for (int j = 0; j < NW; j++) {
            const int64_t n = n0 + 16 * j + 4 * (lane >> 4);
            if (n < a.n) i8_store4<T>(a, m, n, acc[mb][j], sx, sw[j], b[j]);
        }
    }
}

template <class T>
static int i8_matmul(const I8MatArgs &a, hipStream_t s) {
    auto go = [&](auto kernel, int mb, int nw) {
        const int64_t tm = (a.m + 16 * mb - 1) / (16 * mb), tn = (a.n + 64 * nw - 1) / (64 * nw);
        hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(256), 2 * 16 * mb * I8_STEP, s, a, (int)tm);
        return check_launch("k_i8_tile");
    };
    if (a.m <= 16) return go(k_i8_tile<T, 1, 1>, 1, 1);
    if (a.m <= 128) return go(k_i8_tile<T, 4, 1>, 4, 1);
    return go(k_i8_tile<T, 8, 4>, 8, 4);
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
    CW_REQUIRE(ldy >= n, "i8_matmul: rows of y of %lld %lld apart", (long long)n, (long long)ldy);
    if (m == 0) return CW_OK;
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
    a.rb = (int)i8_row_bytes(k);
    a.y = y;
    a.ldy = ldy;
    hipStream_t s = (hipStream_t)stream;
    if (ydtype == CW_F16) return i8_matmul<_Float16>(a, s);
    if (ydtype == CW_BF16) return i8_matmul<bf16_t>(a, s);
    return i8_matmul<float>(a, s);
}

}  // extern "C"
