// The product of rows of e4m3 codes on the matrix cores, with scales of 128 columns of k.
#pragma once
#include "cw_f8.h"
#include "cw_f8_dev.h"
#include "cw_gmm_dev.h"

namespace cw {

typedef int i32x8v __attribute__((ext_vector_type(8)));

// A lane's 32 codes of a row of the step, and the product of two rows' on the matrix cores: lane l gives the codes of weight row
// l % 16 (A) and of activation row l % 16 (B), any 32 of the 128 of the step that both operands share (here the 16 from 16 (l / 16)
// and the 16 from 64 + 16 (l / 16)), and gets weight rows 4 (l / 16) + 0..3 of activation row l % 16: four neighbouring outputs
// of one row. The sum of the step alone: what it is multiplied with, the scales of these 128 columns, changes with the step.
//
// v_mfma_f32_16x16x128_f8f6f4 takes the codes as they are. It adds the products of 8 neighbouring codes with no more than 18 bits below the
// largest of them (measured on this part: 2^16 + 2^-2 is kept, 2^16 + 2^-3 is 2^16), and those sums in f32: 1.4e-5 of a result of
// random codes, a hundredth of bf16's rounding and a twelfth of f16's. EXACT: as f16, which holds every e4m3 value, at half the
// rate: each product exact and added in f32 (4e-7), for results in f32 and for hidden values whose codes hang on them.
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

// A step's sum p, |p| below 2^25, times the scales sx and sw, onto acc: in f32, where the scales are usual ones, zero or from 2^-63 to
// 2^63 (their product is zero or a normal number). Others, which a program's own codes may have: by the fraction and the exponent of
// the product in 64 bits, so that nothing but the result leaves f32's range. One formula for a row, whatever the rows beside it are.
__device__ __forceinline__ bool f8_usual(float s) {
    const uint32_t u = __float_as_uint(s) & 0x7FFFFFFFu;
    return u == 0 || (u >= 64u << 23 && u <= 190u << 23);
}
struct F8Scale {
    float s;  // the product, or its fraction
    int e;
    bool usual;
    __device__ __forceinline__ F8Scale(float sx, float sw) {
        usual = f8_usual(sx) && f8_usual(sw);
        const double d = (double)sx * sw;
        s = usual ? sx * sw : (float)__builtin_amdgcn_frexp_mant(d);
        e = usual ? 0 : __builtin_amdgcn_frexp_exp(d);
    }
    __device__ __forceinline__ float add(float p, float acc) const { return usual ? fmaf(p, s, acc) : acc + ldexpf(p * s, e); }
};

// four neighbouring outputs
template <class T>
__device__ __forceinline__ void f8_store4(T *y, int valid, f32x4 v, const float (&b)[4]) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = v[i] + b[i];
    store_row<4>(y, valid, f);
}

}  // namespace cw
