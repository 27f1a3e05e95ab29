// What the products of 8-bit block-scaled operands share.
//
// Codes are e4m3 (a sign, four bits of exponent with bias 7, three of mantissa; largest 448, one NaN, no infinity).  A matrix
// [N, K] has one fp32 scale for each block of 128 x 128.  It is laid out block by block, [blocks of rows, blocks of columns, 128, 128], padded with
// zero codes to whole blocks, so that a step's 16 KB lie side by side in memory; its scales are [blocks of rows, blocks of columns].  In a matrix of (gate, up) row
// pairs (row 2i = gate i, 2i + 1 = up i) the scales' rows alternate likewise: row 2j of them is the gate's block j, 2j + 1 the up's.
// Rows x [M, K] have one power of two for each run of 128 columns; their scales lie [runs, M rounded up to 4].
#pragma once

#include <cuda_fp16.h>

#include "moe.cuh"
#include "tcgen05.cuh"

namespace tib {

constexpr int kBlk = 128;

// the row of the scales that feature f has
__host__ __device__ __forceinline__ int bs_scale_row(int f, int pairs) { return pairs ? ((f >> 8) << 1) | (f & 1) : f >> 7; }

// The scale of a run whose largest absolute value has these bits, and what its numbers are multiplied by: 2^p and 2^-p with p the smallest integer, at
// least -126, for which the largest is at most 448 * 2^p (448 = 1.75 * 2^8: the exponent less 8, one more where the mantissa is above 1.75); 1 for a run
// of zeros; NaN where the largest is an infinity or a NaN, so that such a row shows in every output.  A power of two divides without rounding, so that codes are
// the same on any machine, and multiplies another scale without rounding (but see BsFar).  What it costs: with (largest / 448) as its scale a run's largest number is
// a code exactly, here it is rounded like any other.  Relative rms error of rows and of products with them, this / that: Gaussian rows 0.0266 / 0.0257,
// silu(g) u of Gaussian ones 0.0265 / 0.0226, rows with one column in a hundred 20 times as large 0.0266 / 0.016.
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

// The scale of a (row, run) and (block, run) is s S, s = 2^p: exact where it is a normal number (or s is at least 1), which is all but everywhere.  Elsewhere the
// sum v of the run's products, 0 or of a size from 2^-18 to 2^25, may still have a share v s S that is a normal number while s S is none.  Such a scale is "far".
// The kernels' loops only notice that a row's s is outside of what the matrix's scales keep normal (from `low` to `high`); behind their tiles the
// outputs with a far scale are made again, by themselves.  No other output changes: a row's bits are its own.  (Shares of far scales made inside the loops cost
// every call 1 to 13 %, a look at the sums as they are finished 1 to 45 %; this costs 0.1 us of 5 to 14 at few rows, nothing at many, and a call whose rows are
// all of 2^-125 milliseconds: 1.4 for 8 rows 4,096 -> 4,096, 23 for 2,048 rows 4,096 -> 6,144.)
struct BsFar {
  float low, high;
  __device__ __forceinline__ bool outside(float s) const { return s < low || s > high; }      // (a NaN is not)
};
__device__ __forceinline__ bool bs_is_far(float s, float s_of_block) {
  const float block = fabsf(s_of_block), product = s * block;
  return product < fminf(block, 0x1p-126f) || (product > 3.402823466e38f && block < INFINITY);      // (a NaN is not)
}

// The sum of 16 products of codes.
__device__ __forceinline__ float bs_dot16(uint4 a, uint4 b) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t p, q;      // (a code is a half without rounding)
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p) : "h"((uint16_t)(x[i >> 1] >> (16 * (i & 1)))));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(q) : "h"((uint16_t)(y[i >> 1] >> (16 * (i & 1)))));
    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&p)), v = __half22float2(*reinterpret_cast<const __half2*>(&q));
    sum = fmaf(u.x, v.x, fmaf(u.y, v.y, sum));
  }
  return sum;
}

// A row of x (codes, TX uint8_t, with scales `lds` apart; or as it is) and the matrix it meets.
template <typename TX> struct BsApart {
  const TX* x;
  const float* x_scales;
  int64_t lds;
  const unsigned char* w;      // the expert's blocks
  const float* w_scales;       // and their scales
  int pairs, runs, K, act;
  float row_scale, limit, alpha;

  __device__ float run_scale(int b, float& inverse) const {
    if constexpr (sizeof(TX) == 1) return x_scales[(size_t)b * lds];
    else {
      uint32_t largest = 0;
      float scale;
#pragma unroll 1
      for (int i = 0; i < kBlk; i += 16) {
        uint4 raw[sizeof(TX)];
        bs_ask16<TX, false>(x + b * kBlk + i, K - b * kBlk - i, raw);
        largest = max(largest, bs_largest16<TX>(raw));
      }
      bs_run_scale(largest, scale, inverse);
      return scale;
    }
  }
  __device__ bool far(int f) const {      // whether feature f's sum has a far scale
    const float* ws = w_scales + (size_t)bs_scale_row(f, pairs) * runs;
    float inverse;
    bool far = false;
    for (int b = 0; b < runs; ++b) {
      const float s = run_scale(b, inverse);
      if (isnan(s)) return false;         // (the row's outputs are NaN)
      far = far || bs_is_far(s, ws[b]);
    }
    return far;
  }
  // By one thread, 16 columns at a time.  A far scale's share is made in two steps, s shifted by 2^64 (without rounding) and the share shifted back:
  // v (s 2^64 S) 2^-64 where S is below 1 and s S too small, v (s 2^-64 S) 2^64 where it is too large (s is at most 2^120: that takes an S of 2^8).
  __device__ float sum(int f) const {
    const float* ws = w_scales + (size_t)bs_scale_row(f, pairs) * runs;
    float inverse = 0.f, sum = 0.f;
    const unsigned char* codes = w + ((size_t)(f >> 7) * runs * kBlk + (f & 127)) * kBlk;
#pragma unroll 1
    for (int b = 0; b < runs; ++b, codes += kBlk * kBlk) {
      const float s = run_scale(b, inverse), block = ws[b];
      float v = 0.f;
#pragma unroll 2
      for (int i = 0; i < kBlk; i += 16) {
        const uint4 wc = *reinterpret_cast<const uint4*>(codes + i);
        if constexpr (sizeof(TX) == 1) v += bs_dot16(*reinterpret_cast<const uint4*>(x + b * kBlk + i), wc);
        else {
          uint4 raw[sizeof(TX)];
          bs_ask16<TX, false>(x + b * kBlk + i, K - b * kBlk - i, raw);
          v += bs_dot16(bs_codes16<TX>(raw, inverse), wc);
        }
      }
      if (bs_is_far(s, block)) {
        const bool small = fabsf(block) < 1.f;
        // (a shifted scale beyond the range: v is 0, or its share an infinity either way)
        const float shifted = fminf(fmaxf(s * (small ? 0x1p64f : 0x1p-64f) * block, -3.402823466e38f), 3.402823466e38f);
        sum = fmaf(v * shifted, small ? 0x1p-64f : 0x1p64f, sum);
      } else {
        sum = fmaf(v, s * block, sum);
      }
    }
    return sum * row_scale;
  }
};
// The row's output o, if it has a far scale, to y.  (Not inline: it is never in a hurry, and the kernels' registers are not for it.)
template <typename TX, typename TO>
__device__ __noinline__ void bs_output_apart(const BsApart<TX>& a, int o, TO* __restrict__ y) {
  const int gated = moe_act_gated(a.act) ? 1 : 0;
  if (!a.far(o << gated) && !(gated && a.far((o << gated) + 1))) return;
  const float g = a.sum(o << gated), u = gated ? a.sum((o << gated) + 1) : 0.f;
  float v = g;
  switch (a.act) {
    case MOE_ACT_RELU2: v = bs_act<MOE_ACT_RELU2>(g); break;
    case MOE_ACT_SILU: v = bs_act<MOE_ACT_SILU>(g); break;
    case MOE_ACT_GELU: v = bs_act<MOE_ACT_GELU>(g); break;
    case MOE_ACT_GLU_CLAMP: v = bs_gated<MOE_ACT_GLU_CLAMP>(g, u, a.limit, a.alpha); break;
    case MOE_ACT_SWIGLU: v = bs_gated<MOE_ACT_SWIGLU>(g, u, a.limit, a.alpha); break;
  }
  y[o] = from_f32<TO>(v);
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
                             const float* row_scale, float far_low, float far_high, int* error_word, cudaStream_t stream);
int tib_block_scaled_tcgen05_plan(int codes, int M, int N, int K, int experts, int* plan);
int tib_block_scaled_2cta_experts();
int tib_block_scaled_2cta_plan(int M, int N, int K, int experts, int* plan);
int tib_block_scaled_2cta(const void* x, const float* x_scales, int64_t lds, const void* w, const float* w_scales, int scale_rows, int pairs,
                          void* out, int out_dtype, int64_t ldo, int M, int N, int K, const int* offsets, const int* order, int experts, int act,
                          float limit, float alpha, const float* row_scale, float far_low, float far_high, int* error_word, cudaStream_t stream);
}
