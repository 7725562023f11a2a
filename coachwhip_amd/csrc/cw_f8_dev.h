// Device code shared by the 8-bit float kernels. e4m3 (OCP): 1 sign, 4 exponent, 3 fraction bits, largest value 448, no infinity.
#pragma once
#include "cw_i8_dev.h"

namespace cw {

typedef float f32x2v __attribute__((ext_vector_type(2)));

// The largest magnitude over 16 neighbouring lanes, as its bits (infinities and NaNs above all finite values), in each of them
__device__ __forceinline__ uint32_t max16_u(uint32_t v) {
    v = max(v, dpp_u<0xB1>(v));
    v = max(v, dpp_u<0x4E>(v));
    v = max(v, dpp_u<0x141>(v));
    return max(v, dpp_u<0x140>(v));
}

// How a group of 128 values whose largest magnitude is a (its bits) becomes codes: scale = a / 448 rounded to f32 and code =
// 448 y / a, rounded to f32 and then to the nearest e4m3 (ties to even). The factor 448 / a and its product with y are in 64 bits:
// a quotient that lies on the border between two codes comes out on it. A group with a value that is not finite gets the scale NaN
// and zero codes, a group of zeros the scale 0.
struct F8Group {
    float scale;
    double factor;
    __device__ __forceinline__ F8Group(uint32_t bits) {
        const double a = __uint_as_float(bits);
        const bool fine = bits < 0x7F800000u;
        double r = __builtin_amdgcn_rcp(a);  // (a of zero: infinite, not used) two Newton steps: 2^-52
        r = fma(fma(-a, r, 1.0), r, r);
        r = fma(fma(-a, r, 1.0), r, r);
        factor = fine && bits ? 448.0 * r : 0.0;
        scale = fine ? (float)(a * (1.0 / 448.0)) : __int_as_float(0x7fc00000);
    }
    __device__ __forceinline__ float quotient(float y) const { return factor != 0.0 ? (float)((double)y * factor) : 0.f; }
};
// four codes, the first in the low byte
__device__ __forceinline__ uint32_t f8_codes4(float a, float b, float c, float d) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
__device__ __forceinline__ uint2 f8_codes8(const F8Group &g, const float (&y)[8]) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = g.quotient(y[i]);
    return make_uint2(f8_codes4(t[0], t[1], t[2], t[3]), f8_codes4(t[4], t[5], t[6], t[7]));
}
__device__ __forceinline__ void f8_values4(uint32_t q, float (&v)[4]) {
    const f32x2v lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
    v[0] = lo[0];
    v[1] = lo[1];
    v[2] = hi[0];
    v[3] = hi[1];
}

}  // namespace cw
