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

}  // namespace cw
