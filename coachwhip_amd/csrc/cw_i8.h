// Internal interface of the 8-bit integer path (cw_i8.hip, cw_i8_gemm.hip, cw_i8_moe.hip): rows of
// ceil(k / 128) * 128 codes (zeros past k) with an f32 scale each.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cw_common.h"

namespace cw {

inline int64_t i8_row_bytes(int64_t k) { return (k + 127) / 128 * 128; }
inline bool i8_float_type(int dtype) { return dtype == CW_F32 || dtype == CW_F16 || dtype == CW_BF16; }
inline bool i8_aligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// codes and scales of `rows` rows of k floats, ldx floats apart
int i8_quantize_f32(const float *x, int64_t rows, int64_t k, int64_t ldx, int8_t *q, float *scale, hipStream_t s);

}  // namespace cw
