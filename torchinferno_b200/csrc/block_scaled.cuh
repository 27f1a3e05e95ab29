// What the products of 8-bit block-scaled operands share.
//
// Codes are e4m3 (a sign, four bits of exponent with bias 7, three of mantissa; largest 448, one NaN, no infinity).  A matrix
// [N, K] has one fp32 scale for each block of 128 x 128.  It is laid out block by block, [blocks of rows, blocks of columns, 128, 128], padded with
// zero codes to whole blocks, so that a step's 16 KB lie side by side in memory; its scales are [blocks of rows, blocks of columns].  In a matrix of (gate, up) row
// pairs (row 2i = gate i, 2i + 1 = up i) the scales' rows alternate likewise: row 2j of them is the gate's block j, 2j + 1 the up's.
// Rows x [M, K] have one power of two for each run of 128 columns; their scales lie [runs, M rounded up to 4].
#pragma once

#include "moe.cuh"
#include "tcgen05.cuh"

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

// 1 / (1 + e^-x) with the approximate exponential and reciprocal: a relative error of a few 2^-23 (1 + |x|).  Where e^-x is beyond 2^126, at x under
// -87, it is 0.
__device__ __forceinline__ float bs_sigmoid(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-x)));
  return r;
}

// The experts' activations (moe.cuh) with this sigmoid; a NaN stays one (a minimum or maximum of floats would pass over it).
template <int ACT> __device__ __forceinline__ float bs_act(float v) {
  if (ACT == MOE_ACT_RELU2) return v < 0.f ? 0.f : v * v;
  if (ACT == MOE_ACT_SILU) return v * bs_sigmoid(v);
  return ACT == MOE_ACT_GELU ? gelu_erf(v) : v;
}
template <int ACT> __device__ __forceinline__ float bs_gated(float g, float u, float limit, float alpha) {
  if (ACT == MOE_ACT_SWIGLU) return g * bs_sigmoid(g) * u;
  g = g > limit ? limit : g;
  u = u > limit ? limit : u < -limit ? -limit : u;
  return g * bs_sigmoid(alpha * g) * (u + 1.f);
}

// Rows sorted by expert, kept within what there is: expert e's first row and the one behind its last, and the pair that sorted row `at` is.
__device__ __forceinline__ int bs_offset(const int* __restrict__ offsets, int e, int M) { return min(max(offsets[e], 0), M); }
__device__ __forceinline__ int bs_pair(const int* __restrict__ order, int at, int M) { return min(max(order[at], 0), M - 1); }

// two floats to two codes (the first in the lower byte), to nearest, ties to even; a NaN stays one
__device__ __forceinline__ uint32_t bs_codes2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t bs_codes4(float a, float b, float c, float d) { return bs_codes2(a, b) | (bs_codes2(c, d) << 16); }

// Sixteen numbers of a row, those from the n-th on zero, as they lie in memory (VEC: p is 16-byte aligned), and as floats.  (Two steps, so that a
// load may be on its way while others are worked on.)
template <typename T, bool VEC> __device__ __forceinline__ void bs_ask16(const T* p, int n, uint4 (&raw)[sizeof(T)]) {
  constexpr int kPer = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) {
    if (VEC && n >= (i + 1) * kPer) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    else {
      T piece[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) piece[j] = i * kPer + j < n ? p[i * kPer + j] : from_f32<T>(0.f);
      raw[i] = *reinterpret_cast<const uint4*>(piece);
    }
  }
}
template <typename T> __device__ __forceinline__ void bs_floats16(const uint4 (&raw)[sizeof(T)], float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) {
        v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
        v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      } else v[4 * i + j] = __uint_as_float(w[j]);
    }
  }
}

// The bits of the largest absolute value of sixteen numbers: of bf16, two at a time by their halves of a word.
template <typename T> __device__ __forceinline__ uint32_t bs_largest16(const uint4 (&raw)[sizeof(T)]) {
  uint32_t w[4 * sizeof(T)];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) {
    w[4 * i] = raw[i].x; w[4 * i + 1] = raw[i].y; w[4 * i + 2] = raw[i].z; w[4 * i + 3] = raw[i].w;
  }
  constexpr uint32_t kMask = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
#pragma unroll
  for (int i = 0; i < 4 * (int)sizeof(T); ++i) w[i] &= kMask;
#pragma unroll
  for (int n = 2 * sizeof(T); n > 0; n >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) w[i] = sizeof(T) == 2 ? __vmaxu2(w[i], w[i + n]) : max(w[i], w[i + n]);
  return sizeof(T) == 2 ? max(w[0] << 16, w[0] & 0xffff0000u) : w[0];
}
// Sixteen codes of sixteen numbers times `inverse`.
template <typename T> __device__ __forceinline__ uint4 bs_codes16(const uint4 (&raw)[sizeof(T)], float inverse) {
  float v[16];
  bs_floats16<T>(raw, v);
  const f32x2 inverse2 = f2_pack(inverse, inverse);
#pragma unroll
  for (int j = 0; j < 16; j += 2) f2_unpack(f2_mul(f2_pack(v[j], v[j + 1]), inverse2), v[j], v[j + 1]);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = bs_codes4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Codes [rows, bytes a row], read in boxes of box_rows x 128 with 128-byte swizzle.
static inline int bs_make_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t bytes, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return TIB_E_ARG;
  const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)bytes};
  const cuuint32_t box[2] = {128u, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TIB_OK : TIB_E_ARG;
}

}  // namespace tib

// What a product of block-scaled operands is made of (block_scaled.cu, block_scaled_tcgen05.cu, block_scaled_2cta.cu).
extern "C" {
int tib_quantize_rows(const void* x, int x_dtype, int64_t ldx, void* codes, int64_t ldc, float* scales, int64_t lds, int rows, int K,
                      const int* order, int top, const int* sorted, int x_rows, cudaStream_t stream);
int tib_block_scaled_tcgen05(const void* x, int x_dtype, int64_t ldx, int x_rows, const float* x_scales, int64_t lds, const void* w,
                             const float* w_scales, int scale_rows, int pairs, void* y, int y_dtype, int64_t ldy, int M, int N, int K,
                             const int* offsets, const int* order, int experts, int top, int x_by_pair, int act, float limit, float alpha,
                             const float* row_scale, int* error_word, cudaStream_t stream);
int tib_block_scaled_2cta_experts();
int tib_block_scaled_2cta(const void* x, const float* x_scales, int64_t lds, const void* w, const float* w_scales, int scale_rows, int pairs,
                          void* out, int out_dtype, int64_t ldo, int M, int N, int K, const int* offsets, const int* order, int experts, int act,
                          float limit, float alpha, const float* row_scale, int* error_word, cudaStream_t stream);
}
