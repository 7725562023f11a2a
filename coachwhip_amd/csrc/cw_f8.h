// Internal interface of the 8-bit float path (cw_f8.hip, cw_f8_gemm.hip, cw_f8_moe.hip): rows of ceil(k / 128) * 128 e4m3 codes
// (zeros past k), scales of 128 columns (rows) or of 128 x 128 (matrices).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cw_common.h"

namespace cw {

constexpr int F8_BLOCK = 128;  // columns of a scale, and rows of a matrix's
inline int64_t f8_blocks(int64_t k) { return (k + F8_BLOCK - 1) / F8_BLOCK; }
inline int64_t f8_row_bytes(int64_t k) { return f8_blocks(k) * F8_BLOCK; }
inline bool f8_float_type(int dtype) { return dtype == CW_F32 || dtype == CW_F16 || dtype == CW_BF16; }
inline bool f8_aligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// cw_f8_matmul_experts; f32 results with exact products, or with the 8-bit instruction's (f16's are always exact, bf16's never)
int f8_matmul_experts(const uint8_t *w, int64_t w_stride, const float *w_scale, int n_experts, int64_t n, int64_t k, const uint8_t *x,
                      const float *x_scale, int64_t m, const int32_t *order, int K, int64_t picks, const void *tiles, const float *bias, int ydtype,
                      void *y, int64_t ldy, bool exact, hipStream_t s);

}  // namespace cw
