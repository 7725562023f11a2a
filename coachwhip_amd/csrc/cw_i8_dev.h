// Device code shared by the 8-bit integer kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "cw_wave.h"

namespace cw {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------ 16- and 32-bit floats

struct bf16_t { uint16_t b; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((uint32_t)v.b << 16); }
// to the nearest, ties to even; a NaN stays one
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float v) { return (_Float16)v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) { return __builtin_bit_cast(bf16_t, (__bf16)v); }

// N values from p, which may be at any address of its type: one wide load (the target takes unaligned ones)
// where all N are inside the row, else the `valid` first ones, zeros after them
template <int N, class T>
__device__ __forceinline__ void load_row(const T *p, int valid, float (&v)[N]) {
    T t[N];
    if (valid >= N) {
        memcpy(t, p, sizeof t);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = to_f32(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = i < valid ? to_f32(p[i]) : 0.f;
    }
}
template <int N, class T>
__device__ __forceinline__ void store_row(T *p, int valid, const float (&v)[N]) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = from_f32<T>(v[i]);
    if (valid >= N) {
        memcpy(p, t, sizeof t);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < valid) p[i] = t[i];
    }
}

// ------------------------------------------------------------------------------ reductions in 64 bits

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = dpp_u<CTRL>((uint32_t)u), hi = dpp_u<CTRL>((uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
__device__ __forceinline__ double readlane_d(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
__device__ __forceinline__ double wave_sum_d(double v) {
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    v += dpp_d<0x140>(v);
    return (readlane_d(v, 0) + readlane_d(v, 16)) + (readlane_d(v, 32) + readlane_d(v, 48));
}
__device__ __forceinline__ double wave_max_d(double v) {
    v = fmax(v, dpp_d<0xB1>(v));
    v = fmax(v, dpp_d<0x4E>(v));
    v = fmax(v, dpp_d<0x141>(v));
    v = fmax(v, dpp_d<0x140>(v));
    return fmax(fmax(readlane_d(v, 0), readlane_d(v, 16)), fmax(readlane_d(v, 32), readlane_d(v, 48)));
}

// ------------------------------------------------------------------------------ codes

// The code of y at inv = 127 / max|y|: y inv rounded to the nearest integer by one fma, whose addend
// 1.5 * 2^52 leaves it in the low bits of the sum (two's complement).
__device__ __forceinline__ uint32_t code(double y, double inv) {
    return (uint32_t)__builtin_bit_cast(uint64_t, fma(y, inv, 6755399441055744.0)) & 0xFFu;
}
__device__ __forceinline__ uint32_t codes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return a | b << 8 | c << 16 | d << 24; }

// An integer sum times its two scales (sx sw: their product in 64 bits, exact), plus b. In 64 bits: a product of two f32 scales
// leaves f32's normal range where the result does not (rows with a largest value of 2^-118 and weights' scales of 5e-4: four
// digits lost; 0 * inf between large ones), in either order. Rounded once, to f32.
__device__ __forceinline__ float scaled(int sum, double sxsw, float b) { return (float)fma((double)sum, sxsw, (double)b); }

// The activation's constants: c1 + c2 = -alpha log2(e) in two f32 terms (alpha 1: silu).
struct Glu {
    int act;
    float limit, c1, c2;
};
inline Glu glu_of(int act, float alpha, float limit) {
    const double c = -1.4426950408889634 * (act == CW_ACT_SILU ? 1.0 : (double)alpha);
    const float c1 = (float)c;
    return Glu{act, limit, c1, (float)(c - (double)c1)};
}
// 1 / (1 + e^(-alpha g)) = 1 / (1 + 2^p), p = g (c1 + c2), with the hardware's 2^x and 1 / x, an ulp each. What p lost when it was
// rounded to f32, lo (up to 2^-17 of a power of two, 30 half steps of the result), comes back to first order, sigma(p + lo) =
// s - s (1 - s) ln2 lo, whose next term is below 2^-35: 6 half steps of f32 at most, whatever g is.
// 12 operations, 6 of them for lo (8,192 rows of 2,880 to codes with the values read back, in a graph: 38.6 us without them, 40.9
// with); the library's exp and a correctly rounded division are about 40. (lo is not finite where g c1 overflows; s is 0 or 1
// there, and the product 0.)
__device__ __forceinline__ float sigmoid(float g, const Glu &a) {
    const float p = g * a.c1, lo = __builtin_amdgcn_fmed3f(fmaf(g, a.c2, fmaf(g, a.c1, -p)), -1.0f, 1.0f);
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(p));
    return fmaf(fmaf(-s, s, s) * lo, -0.6931471805599453f, s);
}
// h = act(g, u): silu(g) u, or the clamped form of gpt-oss (cw_clamped_swiglu, without its biases)
__device__ __forceinline__ float glu(float g, float u, const Glu &a) {
    if (a.act == CW_ACT_SILU) return g * sigmoid(g, a) * u;
    // (comparisons rather than fminf: a NaN stays one)
    g = g > a.limit ? a.limit : g;
    u = u > a.limit ? a.limit : u < -a.limit ? -a.limit : u;
    return (u + 1.0f) * (g * sigmoid(g, a));
}

// the larger of m and |v|'s bits: ordered as the magnitudes are, infinities and NaNs above all finite ones
__device__ __forceinline__ uint32_t max_bits(uint32_t m, float v) { return max(m, __float_as_uint(v) & 0x7FFFFFFFu); }
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
    v = max(v, dpp_u<0xB1>(v));
    v = max(v, dpp_u<0x4E>(v));
    v = max(v, dpp_u<0x141>(v));
    v = max(v, dpp_u<0x140>(v));
    return max(max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
               max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

}  // namespace cw
