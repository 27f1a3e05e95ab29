// What the products of 8-bit block-scaled operands share.
//
// Codes are e4m3 (a sign, four bits of exponent with bias 7, three of mantissa; largest 448, one NaN, no infinity).  A matrix
// [N, K] has one fp32 scale for each block of 128 x 128; its rows are padded with zero codes to whole runs of 128 columns when it is laid
// out (so every row starts on a 128-byte boundary), its scales are [blocks of rows, blocks of columns].  In a matrix of (gate, up) row
// pairs (row 2i = gate i, 2i + 1 = up i) the scales' rows alternate likewise: row 2j of them is the gate's block j, 2j + 1 the up's.
// Rows x [M, K] have one power of two for each run of 128 columns; their scales lie [runs, M rounded up to 4].
#pragma once

#include "common.cuh"
#include "moe.cuh"

namespace tib {

constexpr int kBlk = 128;

// the row of the scales that feature f has
__host__ __device__ __forceinline__ int bs_scale_row(int f, int pairs) { return pairs ? ((f >> 8) << 1) | (f & 1) : f >> 7; }

// The scale of a run whose largest absolute value has these bits, and what its numbers are multiplied by: 2^p and 2^-p with p the smallest integer, at
// least -126, for which the largest is at most 448 * 2^p (448 = 1.75 * 2^8: the exponent less 8, one more where the mantissa is above 1.75); 1 for a run
// of zeros; NaN where the largest is an infinity or a NaN, so that such a row shows in every output.  A power of two costs a float format no
// precision, divides without rounding and multiplies another scale without rounding.
__device__ __forceinline__ void bs_run_scale(uint32_t largest, float& scale, float& inverse) {
  int p = (int)(largest >> 23) - 127 - 8 + ((largest & 0x7fffffu) > 0x600000u);
  p = p < -126 ? -126 : p;
  if (largest == 0) p = 0;
  scale = __uint_as_float((uint32_t)(p + 127) << 23);
  inverse = __uint_as_float((uint32_t)(127 - p) << 23);
  if (largest >= 0x7f800000u) scale = inverse = __uint_as_float(0x7fc00000u);
}

// two floats to two codes (the first in the lower byte), to nearest, ties to even; a NaN stays one
__device__ __forceinline__ uint32_t bs_codes2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t bs_codes4(float a, float b, float c, float d) { return bs_codes2(a, b) | (bs_codes2(c, d) << 16); }

}  // namespace tib
