// Rows to e4m3 codes with a scale for each 128 columns (gfx950): plain or of a SwiGLU; matrices with a scale for each 128 x 128; and
// codes back to floats.
#include <algorithm>

#include "cw_f8.h"
#include "cw_f8_dev.h"

namespace cw {

struct F8RowsArgs {
    const void *x, *u;  // rows, or gate and up
    int64_t ld, rows;
    uint32_t units;
    int k, blocks, strip;  // strip: rows of a unit strip (16, or all of fewer)
    Glu glu;
    uint8_t *q;
    float *scale;
};

// A unit: 128 columns of a row, 16 lanes of 8 neighbouring values each, so that a unit needs nothing from another wave. Units go
// down a strip of 16 rows before they go on to the next 128 columns: their scales lie side by side. 8,192 rows of bf16: of 4,096 23 us (4.4 TB/s), SwiGLU
// of 2,880 27 to 33 (the activation's and the codes' instructions beside the loads).
template <class T, bool GLU>
__global__ __launch_bounds__(256) void k_rows_f8(F8RowsArgs a) {
    const uint32_t unit = blockIdx.x * 16 + (threadIdx.x >> 4);
    if (unit >= a.units) return;  // (16 lanes at a time; no lane reads across them)
    const uint32_t whole = a.strip * a.blocks, s = unit / whole, in = unit - s * whole;
    const int64_t row0 = (int64_t)s * a.strip;
    const uint32_t height = (uint32_t)min((int64_t)a.strip, a.rows - row0);
    const int b = (int)(in / height);
    const int64_t row = row0 + (in - (uint32_t)b * height);
    if (b >= a.blocks) return;  // (the last strip may be lower)
    const int e = F8_BLOCK * b + 8 * (threadIdx.x & 15), valid = a.k - e;
    float y[8];
    load_row<8>((const T *)a.x + row * a.ld + e, valid, y);
    if constexpr (GLU) {
        float u[8];
        load_row<8>((const T *)a.u + row * a.ld + e, valid, u);
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = i < valid ? glu(y[i], u[i], a.glu) : 0.f;
    }
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) bits = max_bits(bits, y[i]);
    const F8Group g(max16_u(bits));
    *(uint2 *)(a.q + row * ((int64_t)a.blocks * F8_BLOCK) + e) = f8_codes8(g, y);
    if ((threadIdx.x & 15) == 0) a.scale[(int64_t)b * a.rows + row] = g.scale;
}

template <class T, bool GLU>
static int rows_launch(const F8RowsArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((k_rows_f8<T, GLU>), dim3((unsigned)((a.units + 15) / 16)), dim3(256), 0, s, a);
    return check_launch("k_rows_f8");
}
template <bool GLU>
static int rows_f8(int dtype, const F8RowsArgs &a, hipStream_t s) {
    if (dtype == CW_F16) return rows_launch<_Float16, GLU>(a, s);
    if (dtype == CW_BF16) return rows_launch<bf16_t, GLU>(a, s);
    return rows_launch<float, GLU>(a, s);
}

// A block of 128 x 128 of a matrix: 16 lanes a row, eight rows a thread, the largest of the block through LDS.
template <class T>
__global__ __launch_bounds__(256) void k_matrix_f8(const T *w, int64_t ld, int n, int k, int blocks, uint8_t *q, float *scale) {
    __shared__ uint32_t top[16];
    const int64_t nb = blockIdx.x / blocks;
    const int kb = (int)(blockIdx.x - nb * blocks), e = F8_BLOCK * kb + 8 * (threadIdx.x & 15), group = threadIdx.x >> 4;
    float y[8][8];
    uint32_t bits = 0;
#pragma unroll
    for (int r = 0; r < 8; r++) {
        const int64_t row = nb * F8_BLOCK + group + 16 * r;
        load_row<8>(w + min(row, (int64_t)n - 1) * ld + e, row < n ? k - e : 0, y[r]);
#pragma unroll
        for (int i = 0; i < 8; i++) bits = max_bits(bits, y[r][i]);
    }
    bits = max16_u(bits);
    if ((threadIdx.x & 15) == 0) top[group] = bits;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) bits = max(bits, top[i]);
    const F8Group g(bits);
#pragma unroll
    for (int r = 0; r < 8; r++) {
        const int64_t row = nb * F8_BLOCK + group + 16 * r;
        if (row < n) *(uint2 *)(q + row * ((int64_t)blocks * F8_BLOCK) + e) = f8_codes8(g, y[r]);
    }
    if (threadIdx.x == 0) scale[blockIdx.x] = g.scale;
}

// 8 codes at a time
template <class T>
__global__ __launch_bounds__(256) void k_dequant_f8(const uint8_t *q, const float *scale, int64_t rows, int k, int cpr, T *out) {
    const int64_t n = rows * cpr, rb = (int64_t)(k + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / cpr;
        const int e = 8 * (int)(i - row * cpr);
        const uint2 p = *(const uint2 *)(q + row * rb + e);
        const float s = scale[(int64_t)(e / F8_BLOCK) * rows + row];
        float lo[4], hi[4], v[8];
        f8_values4(p.x, lo);
        f8_values4(p.y, hi);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = lo[j] * s;
            v[4 + j] = hi[j] * s;
        }
        store_row<8>(out + row * k + e, k - e, v);
    }
}

static int check_rows(const char *what, int dtype, int64_t rows, int64_t k, const void *q, const void *scale) {
    if (!f8_float_type(dtype)) return set_error(CW_ENOTSUP, "%s: type %d (f32, f16 or bf16)", what, dtype);
    CW_REQUIRE(rows >= 0 && rows < (1ll << 31) && k > 0, "%s: %lld rows of %lld", what, (long long)rows, (long long)k);
    if (k > CW_F8_MAX_K) return set_error(CW_ENOTSUP, "%s: rows of %lld above %d", what, (long long)k, CW_F8_MAX_K);
    // (a launch holds fewer than 2^32 threads, 16 of a unit)
    if (rows * f8_blocks(k) >= 1ll << 27) return set_error(CW_ENOTSUP, "%s: %lld rows of %lld", what, (long long)rows, (long long)k);
    CW_REQUIRE(rows == 0 || (q && scale), "%s: null pointer", what);
    CW_REQUIRE(f8_aligned(q, 16), "%s: codes must be 16-byte aligned", what);
    return CW_OK;
}

static F8RowsArgs rows_args(const void *x, int64_t ld, int64_t rows, int64_t k, uint8_t *q, float *scale) {
    F8RowsArgs a = {};
    a.x = x;
    a.ld = ld;
    a.rows = rows;
    a.k = (int)k;
    a.blocks = (int)f8_blocks(k);
    a.strip = (int)std::min<int64_t>(rows, 16);
    a.units = (uint32_t)((rows + a.strip - 1) / a.strip * a.strip * a.blocks);
    a.q = q;
    a.scale = scale;
    return a;
}

}  // namespace cw

using namespace cw;

extern "C" {

int64_t cw_f8_row_bytes(int64_t k) { return k > 0 ? f8_row_bytes(k) : 0; }

int cw_quantize_f8(int dtype, const void *x, int64_t ldx, int64_t rows, int64_t k, uint8_t *q, float *scale, cw_stream_t stream) {
    if (int rc = check_rows("quantize_f8", dtype, rows, k, q, scale)) return rc;
    if (rows == 0) return CW_OK;
    CW_REQUIRE(x && ldx >= k, "quantize_f8: null x, or rows of %lld %lld apart", (long long)k, (long long)ldx);
    return rows_f8<false>(dtype, rows_args(x, ldx, rows, k, q, scale), (hipStream_t)stream);
}

int cw_swiglu_f8(int dtype, const void *g, const void *u, int64_t ld, int64_t rows, int64_t width, int act, float alpha, float limit,
                 uint8_t *q, float *scale, cw_stream_t stream) {
    if (int rc = check_rows("swiglu_f8", dtype, rows, width, q, scale)) return rc;
    CW_REQUIRE(act == CW_ACT_SILU || act == CW_ACT_CLAMPED_SWIGLU, "swiglu_f8: unknown activation %d", act);
    if (rows == 0) return CW_OK;
    CW_REQUIRE(g && u && ld >= width, "swiglu_f8: null pointer, or rows of %lld %lld apart", (long long)width, (long long)ld);
    F8RowsArgs a = rows_args(g, ld, rows, width, q, scale);
    a.u = u;
    a.glu = glu_of(act, alpha, limit);
    return rows_f8<true>(dtype, a, (hipStream_t)stream);
}

int cw_quantize_f8_matrix(int dtype, const void *w, int64_t ldw, int64_t n, int64_t k, uint8_t *q, float *scale, cw_stream_t stream) {
    if (int rc = check_rows("quantize_f8_matrix", dtype, n, k, q, scale)) return rc;
    if (n == 0) return CW_OK;
    CW_REQUIRE(w && ldw >= k, "quantize_f8_matrix: null w, or rows of %lld %lld apart", (long long)k, (long long)ldw);
    const int blocks = (int)f8_blocks(k);
    const dim3 grid((unsigned)(f8_blocks(n) * blocks));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == CW_F16) hipLaunchKernelGGL(k_matrix_f8<_Float16>, grid, dim3(256), 0, s, (const _Float16 *)w, ldw, (int)n, (int)k, blocks, q, scale);
    else if (dtype == CW_BF16) hipLaunchKernelGGL(k_matrix_f8<bf16_t>, grid, dim3(256), 0, s, (const bf16_t *)w, ldw, (int)n, (int)k, blocks, q, scale);
    else hipLaunchKernelGGL(k_matrix_f8<float>, grid, dim3(256), 0, s, (const float *)w, ldw, (int)n, (int)k, blocks, q, scale);
    return check_launch("k_matrix_f8");
}

int cw_dequantize_f8(const uint8_t *q, const float *scale, int64_t rows, int64_t k, int dtype, void *out, cw_stream_t stream) {
    if (int rc = check_rows("dequantize_f8", dtype, rows, k, q, scale)) return rc;
    if (rows == 0) return CW_OK;
    CW_REQUIRE(out, "dequantize_f8: null pointer");
    const int cpr = (int)((k + 7) / 8);
    const dim3 grid((unsigned)std::min<int64_t>((rows * cpr + 255) / 256, 1 << 21));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == CW_F16) hipLaunchKernelGGL(k_dequant_f8<_Float16>, grid, dim3(256), 0, s, q, scale, rows, (int)k, cpr, (_Float16 *)out);
    else if (dtype == CW_BF16) hipLaunchKernelGGL(k_dequant_f8<bf16_t>, grid, dim3(256), 0, s, q, scale, rows, (int)k, cpr, (bf16_t *)out);
    else hipLaunchKernelGGL(k_dequant_f8<float>, grid, dim3(256), 0, s, q, scale, rows, (int)k, cpr, (float *)out);
    return check_launch("k_dequant_f8");
}

}  // extern "C"
