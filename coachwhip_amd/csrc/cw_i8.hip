// Rows to 8-bit codes with a scale each (gfx950): plain, of a SwiGLU, or of an RMS norm with the
// residual's addition; and codes back to floats.
#include "cw_i8.h"
#include "cw_i8_dev.h"

namespace cw {

enum { ROWS_PLAIN = 0, ROWS_GLU = 1, ROWS_NORM = 2 };

struct RowsArgs {
    const void *x, *r;        // plain: x; GLU: gate, up; norm: x, residual (or NULL)
    int64_t ldx, ldr;         // elements between rows
    int64_t rows, row0;       // this launch: rows row0 .. rows - 1
    int k;
    Glu glu;
    const float *w;           // norm
    double eps;
    void *sum;                // norm: x + r (or NULL), rows of k
    float *y;                 // norm: the normalised rows (or NULL), rows of k
    uint8_t *q;               // rows of ceil(k / 128) * 128 codes
    float *scale;
};

// TPR threads per row, each NCH chunks of 8 elements held in registers (chunk c of thread t: elements
// 8 (t + c TPR)..): one pass over the inputs. a = max|y|, scale = a / 127 rounded to f32, code =
// y * 127 / a to the nearest. The norm's mean, factor and products and every code are computed in 64 bits,
// whose vector rate here is half that of 32: a code does not depend on the order of a sum, and the kernel
// stays bound by its bytes. A row with a value that is not finite, or whose scale would not be, gets the scale NaN and
// zero codes; a row of zeros the scale 0. 8,192 rows, bf16: norm of 4,096 50 us (4.7 TB/s), SwiGLU of 2,880 30 (3.9; about 38 vector
// operations a value).
template <class T, int MODE, int TPR, int NCH>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void k_rows_i8(RowsArgs a) {
    constexpr int NT = TPR == 64 ? 256 : TPR, RPB = NT / TPR, WPR = TPR / 64;
    __shared__ double red[2][NT / 64];
    const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR, wave = threadIdx.x / 64;
    const int64_t row = a.row0 + (int64_t)blockIdx.x * RPB + sub;
    if (TPR == 64 && row >= a.rows) return;  // whole waves, and no barrier follows
    const T *x = (const T *)a.x + row * a.ldx, *r = (const T *)a.r + row * a.ldr;
    using V = std::conditional_t<MODE == ROWS_NORM, double, float>;
    V y[NCH][8];
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
        const int e = 8 * (tid + c * TPR), valid = a.k - e;
        float v[8];
        load_row<8>(x + e, valid, v);
        if constexpr (MODE == ROWS_GLU) {
            float u[8];
            load_row<8>(r + e, valid, u);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = i < valid ? glu(v[i], u[i], a.glu) : 0.f;
        }
        if constexpr (MODE == ROWS_NORM) {
            if (a.r) {
                float u[8];
                load_row<8>(r + e, valid, u);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = to_f32(from_f32<T>(v[i] + u[i]));
                if (a.sum && valid > 0) store_row<8>((T *)a.sum + row * a.k + e, valid, v);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fma((double)v[i], (double)v[i], ss);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) y[c][i] = v[i];
    }
    if constexpr (MODE == ROWS_NORM) {
        ss = wave_sum_d(ss);
        if constexpr (WPR > 1) {
            if ((threadIdx.x & 63) == 0) red[0][wave] = ss;
            __syncthreads();
            ss = 0.0;
#pragma unroll
            for (int w = 0; w < WPR; w++) ss += red[0][w];
        }
        const double f = 1.0 / sqrt(ss / a.k + a.eps);
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const int e = 8 * (tid + c * TPR), valid = a.k - e;
            float w[8];  // (loaded here: with the row, its registers cost 8,192 rows of 4,096 50 -> 55 us, and few rows gain nothing)
            load_row<8>(a.w + e, valid, w);
#pragma unroll
            for (int i = 0; i < 8; i++) y[c][i] = y[c][i] * f * w[i];
            if (a.y && valid > 0) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = (float)y[c][i];
                store_row<8>(a.y + row * a.k + e, valid, v);
            }
        }
    }
    // the largest magnitude; a NaN or an infinity makes it infinite
    double m = 0.0;
    if constexpr (MODE == ROWS_NORM) {
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const double v = fabs(y[c][i]);
                m = v <= m ? m : v < INFINITY ? v : INFINITY;
            }
        m = wave_max_d(m);
    } else {
        uint32_t bits = 0;
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) bits = max_bits(bits, y[c][i]);
        bits = wave_max_u(bits);
        m = bits < 0x7F800000u ? (double)__uint_as_float(bits) : (double)INFINITY;
    }
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) red[1][wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; w++) m = fmax(m, red[1][w]);
    }
    const bool fine = m <= 127.0 * (double)__FLT_MAX__, codes = fine && m > 0.0;  // (a norm's values may pass f32's, and so the scale)
    const double inv = codes ? 127.0 / m : 0.0;
    const int rb = (a.k + 127) / 128 * 128;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
        const int e = 8 * (tid + c * TPR);
        if (e >= rb) break;
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = codes ? code(y[c][i], inv) : 0u;
        *(uint2 *)(a.q + row * rb + e) = make_uint2(codes4(q[0], q[1], q[2], q[3]), codes4(q[4], q[5], q[6], q[7]));
    }
    if (tid == 0) a.scale[row] = fine ? (float)(m / 127.0) : __int_as_float(0x7fc00000);
}

template <class T, int MODE>
static int rows_launch(RowsArgs a, hipStream_t s) {
    const int chunks = (a.k + 127) / 128 * 16;
    constexpr int64_t MAX_BLOCKS = 1 << 21;  // (a launch holds fewer than 2^32 threads)
#define CW_ROWS(TPR, NCH) \
    if (chunks <= TPR * NCH) { \
        constexpr int RPB = TPR == 64 ? 4 : 1; \
        for (; a.row0 < a.rows; a.row0 += MAX_BLOCKS * RPB) { \
            const int64_t blocks = (a.rows - a.row0 + RPB - 1) / RPB; \
            hipLaunchKernelGGL((k_rows_i8<T, MODE, TPR, NCH>), dim3((unsigned)(blocks < MAX_BLOCKS ? blocks : MAX_BLOCKS)), \
                               dim3(TPR == 64 ? 256 : TPR), 0, s, a); \
            if (int rc = check_launch("k_rows_i8")) return rc; \
        } \
        return CW_OK; \
    }
    // Threads a row, measured with bf16, norm / SwiGLU / plain, us: 8,192 rows of 512 64 threads 8.9 / 7.5 / 4.6, 128 12.6 / 8.6 /
    // 5.6; 8,192 of 4,096 256 threads 48.5 / 34.9 / 19.2, 128 53.3 / 39.1 / 21.5, 512 57.3 / 39.1 / 21.8; one row of 2,048 256
    // threads 2.9 / 2.9 / 2.4, 64 4.8 / 5.6 / 2.8. Rows of 257 to 384 pieces, for which 256 threads take two pieces each and leave
    // up to half of them empty, norm / SwiGLU with 128 threads and with 256, bf16: 2,176 columns 8,192 rows 30.5 / 26.4 and 35.0 /
    // 28.6, 2,048 rows 10.3 / 9.3 and 12.4 / 10.2, 1,024 rows 7.2 / 7.6 and 7.3 / 6.8, 301 rows 6.1 / 6.2 and 5.2 / 5.0; 3,040 columns
    // 37.3 / 31.6 and 41.1 / 33.3, 11.3 / 10.1 and 13.4 / 11.3, 7.9 / 7.9 and 8.0 / 7.4, 6.0 / 5.9 and 5.2 / 5.0; 2,560 and 2,880 and f16
    // alike. f32 is bound by its bytes: within 3 % either way from 4,096 rows, 128 threads 7 to 11 % faster (norm) at 2,048.
    if constexpr (MODE != ROWS_PLAIN) {
        if (a.rows >= 2048 && chunks > 256) {
            CW_ROWS(128, 3)
        }
    }
    CW_ROWS(64, 1) CW_ROWS(64, 2) CW_ROWS(256, 1) CW_ROWS(256, 2) CW_ROWS(256, 4) CW_ROWS(1024, 2) CW_ROWS(1024, 4)
#undef CW_ROWS
    return set_error(CW_ENOTSUP, "i8 rows: %d columns above %d", a.k, CW_I8_MAX_K);
}

template <int MODE>
static int rows_i8(int dtype, const RowsArgs &a, hipStream_t s) {
    if (dtype == CW_F16) return rows_launch<_Float16, MODE>(a, s);
    if (dtype == CW_BF16) return rows_launch<bf16_t, MODE>(a, s);
    return rows_launch<float, MODE>(a, s);
}

int i8_quantize_f32(const float *x, int64_t rows, int64_t k, int64_t ldx, int8_t *q, float *scale, hipStream_t s) {
    RowsArgs a = {};
    a.x = x;
    a.ldx = ldx;
    a.rows = rows;
    a.k = (int)k;
    a.q = (uint8_t *)q;
    a.scale = scale;
    return rows_i8<ROWS_PLAIN>(CW_F32, a, s);
}

// 8 codes at a time
template <class T>
__global__ __launch_bounds__(256) void k_dequant_i8(const uint8_t *q, const float *scale, int64_t n_chunks, int k, int cpr, T *out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / cpr;
        const int e = 8 * (int)(i - row * cpr);
        const uint2 p = *(const uint2 *)(q + row * ((k + 127) / 128 * 128) + e);
        const float s = scale[row];
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = (float)(int8_t)(p.x >> (8 * j)) * s;
            v[4 + j] = (float)(int8_t)(p.y >> (8 * j)) * s;
        }
        store_row<8>(out + row * k + e, k - e, v);
    }
}

static int check_rows(const char *what, int dtype, int64_t rows, int64_t k, const void *q, const void *scale) {
    if (!i8_float_type(dtype)) return set_error(CW_ENOTSUP, "%s: type %d (f32, f16 or bf16)", what, dtype);
    CW_REQUIRE(rows >= 0 && rows < (1ll << 31) && k > 0, "%s: %lld rows of %lld", what, (long long)rows, (long long)k);
    if (k > CW_I8_MAX_K) return set_error(CW_ENOTSUP, "%s: rows of %lld above %d", what, (long long)k, CW_I8_MAX_K);
    CW_REQUIRE(rows == 0 || (q && scale), "%s: null pointer", what);
    CW_REQUIRE(i8_aligned(q, 16), "%s: codes must be 16-byte aligned", what);
    return CW_OK;
}

}  // namespace cw

using namespace cw;

extern "C" {

int64_t cw_i8_row_bytes(int64_t k) { return k > 0 ? i8_row_bytes(k) : 0; }

int cw_quantize_i8(int dtype, const void *x, int64_t ldx, int64_t rows, int64_t k, int8_t *q, float *scale, cw_stream_t stream) {
    if (int rc = check_rows("quantize_i8", dtype, rows, k, q, scale)) return rc;
    if (rows == 0) return CW_OK;
    CW_REQUIRE(x && ldx >= k, "quantize_i8: null x, or rows of %lld %lld apart", (long long)k, (long long)ldx);
    RowsArgs a = {};
    a.x = x;
    a.ldx = ldx;
    a.rows = rows;
    a.k = (int)k;
    a.q = (uint8_t *)q;
    a.scale = scale;
    return rows_i8<ROWS_PLAIN>(dtype, a, (hipStream_t)stream);
}

int cw_swiglu_i8(int dtype, const void *g, const void *u, int64_t ld, int64_t rows, int64_t width, int act, float alpha, float limit,
                 int8_t *q, float *scale, cw_stream_t stream) {
    if (int rc = check_rows("swiglu_i8", dtype, rows, width, q, scale)) return rc;
    CW_REQUIRE(act == CW_ACT_SILU || act == CW_ACT_CLAMPED_SWIGLU, "swiglu_i8: unknown activation %d", act);
    if (rows == 0) return CW_OK;
    CW_REQUIRE(g && u && ld >= width, "swiglu_i8: null pointer, or rows of %lld %lld apart", (long long)width, (long long)ld);
    RowsArgs a = {};
    a.x = g;
    a.r = u;
    a.ldx = a.ldr = ld;
    a.rows = rows;
    a.k = (int)width;
    a.glu = glu_of(act, alpha, limit);
    a.q = (uint8_t *)q;
    a.scale = scale;
    return rows_i8<ROWS_GLU>(dtype, a, (hipStream_t)stream);
}

int cw_rmsnorm_i8(int dtype, const void *x, int64_t ldx, const void *residual, int64_t ldr, const float *weight, float eps, int64_t rows,
                  int64_t k, void *sum, float *y, int8_t *q, float *scale, cw_stream_t stream) {
    if (int rc = check_rows("rmsnorm_i8", dtype, rows, k, q, scale)) return rc;
    CW_REQUIRE(eps >= 0.f, "rmsnorm_i8: eps %g", (double)eps);
    if (rows == 0) return CW_OK;
    CW_REQUIRE(x && weight && ldx >= k, "rmsnorm_i8: null x or weight, or rows of %lld %lld apart", (long long)k, (long long)ldx);
    CW_REQUIRE(!residual || ldr >= k, "rmsnorm_i8: residual rows of %lld %lld apart", (long long)k, (long long)ldr);
    CW_REQUIRE(!sum || residual, "rmsnorm_i8: a sum without a residual");
    RowsArgs a = {};
    a.x = x;
    a.r = residual;
    a.ldx = ldx;
    a.ldr = ldr;
    a.rows = rows;
    a.k = (int)k;
    a.w = weight;
    a.eps = eps;
    a.sum = sum;
    a.y = y;
    a.q = (uint8_t *)q;
    a.scale = scale;
    return rows_i8<ROWS_NORM>(dtype, a, (hipStream_t)stream);
}

int cw_dequantize_i8(const int8_t *q, const float *scale, int64_t rows, int64_t k, int dtype, void *out, cw_stream_t stream) {
    if (int rc = check_rows("dequantize_i8", dtype, rows, k, q, scale)) return rc;
    if (rows == 0) return CW_OK;
    CW_REQUIRE(out, "dequantize_i8: null pointer");
    const int cpr = (int)((k + 7) / 8);
    const int64_t n = rows * cpr;
    const dim3 grid((unsigned)((n + 255) / 256 < (1 << 21) ? (n + 255) / 256 : (1 << 21)));
    hipStream_t s = (hipStream_t)stream;
    const uint8_t *b = (const uint8_t *)q;
    if (dtype == CW_F16) hipLaunchKernelGGL(k_dequant_i8<_Float16>, grid, dim3(256), 0, s, b, scale, n, (int)k, cpr, (_Float16 *)out);
    else if (dtype == CW_BF16) hipLaunchKernelGGL(k_dequant_i8<bf16_t>, grid, dim3(256), 0, s, b, scale, n, (int)k, cpr, (bf16_t *)out);
    else hipLaunchKernelGGL(k_dequant_i8<float>, grid, dim3(256), 0, s, b, scale, n, (int)k, cpr, (float *)out);
    return check_launch("k_dequant_i8");
}

}  // extern "C"
