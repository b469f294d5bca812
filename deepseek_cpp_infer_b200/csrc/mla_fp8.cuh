// The 8-bit latent cache's row format, shared by the kernels that write and
// read it (layout in include/dsb/dsb.h).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dsb {

constexpr int kPageTok = 64;  // tokens per page

inline bool cache_shape_ok(int R, int P) { return (R == 512 && P == 64) || (R == 128 && P == 32); }

// 2^e for e in [-126, 127].
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }

// Exponent of a row's scale: the least e with amax <= 448 * 2^e (448 = 1.75 *
// 2^8 is the largest e4m3 value), within [-64, 64] so that products of the
// scale with bf16 stay finite; 0 for an all-zero row.
__device__ __forceinline__ int row_scale_exponent(float amax) {
  if (!(amax > 0.0f)) return 0;
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(64, max(-64, e));
}

// Two e4m3 codes as fp16 (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
  return r;
}

}  // namespace dsb
