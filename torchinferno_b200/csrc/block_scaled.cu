// 8-bit block-scaled operands (block_scaled.cuh): rows of activations to codes, and products with matrices of codes.
//
//   quantize_rows         codes and powers of two of rows
//   block_scaled_product  y[m, n] = sum over runs b of s[m, b] S[n's block, b] (sum over the run of x[m, k] w[n, k]), plain or for rows
//                         sorted by expert, with the experts' activations
#include "block_scaled.cuh"

namespace tib {

// ----------------------------------------------------------- rows to codes
// Eight lanes take a run of 128 columns, 16 columns each: their largest absolute value by its bits as an integer (a NaN is then the
// largest of all, where a maximum of floats would pass over it), a butterfly of three steps, one multiplication and one
// conversion a number.  A block takes eight rows and four runs of each, so that the scales of a run, which lie row after row, are written 32 bytes
// at a time.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* p, int n, float (&v)[16]) {
  if constexpr (VEC) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) {
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (n >= (i + 1) * kPer) raw = reinterpret_cast<const uint4*>(p)[i];
      else if (n > i * kPer) {
        T piece[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) piece[j] = i * kPer + j < n ? p[i * kPer + j] : from_f32<T>(0.f);
        raw = *reinterpret_cast<const uint4*>(piece);
      }
      if constexpr (sizeof(T) == 2) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
          v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      } else {
        v[4 * i] = __uint_as_float(raw.x); v[4 * i + 1] = __uint_as_float(raw.y);
        v[4 * i + 2] = __uint_as_float(raw.z); v[4 * i + 3] = __uint_as_float(raw.w);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = j < n ? to_f32(p[j]) : 0.f;
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scales,
                     int64_t lds, int rows, int K, int runs) {
  pdl_wait();
  pdl_trigger();
  // thread = (row of 8, run of 4, eighth of the run)
  const int groups = (runs + 3) >> 2, row8 = blockIdx.x / groups;
  const int eighth = threadIdx.x & 7, row = row8 * 8 + (threadIdx.x >> 5), run = (blockIdx.x - row8 * groups) * 4 + ((threadIdx.x >> 3) & 3);
  const bool in = row < rows && run < runs;
  const int col = run * kBlk + eighth * 16;
  float v[16];
  load16<T, VEC>(x + (size_t)(in ? row : 0) * ldx + (in ? col : 0), in ? K - col : 0, v);
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) largest = max(largest, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  float scale, inverse;
  bs_run_scale(largest, scale, inverse);
  if (!in) return;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = bs_codes4(v[4 * j] * inverse, v[4 * j + 1] * inverse, v[4 * j + 2] * inverse, v[4 * j + 3] * inverse);
  *reinterpret_cast<uint4*>(codes + (size_t)row * ldc + col) = make_uint4(w[0], w[1], w[2], w[3]);
  if (eighth == 0) scales[(size_t)run * lds + row] = scale;
}

// ----------------------------------------------------------- products on fp32 multiply-adds
struct BsProduct {
  const uint8_t* x;            // codes [rows, runs * 128]
  const float* x_scales;       // [runs, lds]
  int64_t lds;
  const uint8_t* w;            // codes [experts, N, runs * 128]
  const float* w_scales;       // [experts, scale rows, runs]
  int scale_rows, pairs;
  int M, N, runs;
  const int* offsets;          // [experts + 1], or null: one matrix, all rows
  const int* order;
  int experts, top, x_by_pair;
  MoeEpilogue ep;
};

__device__ __forceinline__ float code_value(uint8_t c) {
  const int e = (c >> 3) & 15, m = c & 7;
  if ((c & 0x7f) == 0x7f) return __uint_as_float(0x7fc00000u);
  const float v = e ? __uint_as_float((uint32_t)(e + 120) << 23 | (uint32_t)m << 20) : (float)m * 0.001953125f;
  return c & 0x80 ? -v : v;
}

template <typename TO>
__global__ void __launch_bounds__(256)
block_scaled_product_kernel(const BsProduct a, TO* __restrict__ y, int64_t ldy) {
  constexpr int TM = 32, TN = 64;
  __shared__ float xs[TM][kBlk + 1];
  __shared__ float ws[TN][33];
  __shared__ float out[TM][TN + 1];
  pdl_wait();
  int expert = 0, first = 0, rows = a.M, tile = blockIdx.y;
  if (a.offsets) {
    for (expert = 0; expert < a.experts; ++expert) {
      first = a.offsets[expert];
      rows = a.offsets[expert + 1] - first;
      const int tiles = (rows + TM - 1) / TM;
      if (tile < tiles) break;
      tile -= tiles;
    }
    if (expert == a.experts) return;
  }
  const int m0 = tile * TM, n0 = blockIdx.x * TN, ld = a.runs * kBlk;
  const uint8_t* w = a.w + (size_t)expert * a.N * ld;
  const float* w_scales = a.w_scales + (size_t)expert * a.scale_rows * a.runs;
  auto source = [&](int r) { return a.offsets ? (a.x_by_pair ? a.order[first + r] / a.top : first + r) : r; };
  const int tm = threadIdx.x >> 4, tn = threadIdx.x & 15;      // rows 2 tm, 2 tm + 1; features tn + 16 j
  float total[2][4] = {};
  for (int b = 0; b < a.runs; ++b) {
    float part[2][4] = {};
    __syncthreads();
    for (int i = threadIdx.x; i < TM * kBlk; i += 256) {
      const int r = i / kBlk, k = i % kBlk;
      xs[r][k] = m0 + r < rows ? code_value(a.x[(size_t)source(m0 + r) * ld + b * kBlk + k]) : 0.f;
    }
    for (int k0 = 0; k0 < kBlk; k0 += 32) {
      __syncthreads();
      for (int i = threadIdx.x; i < TN * 32; i += 256) {
        const int f = i / 32, k = i % 32;
        ws[f][k] = n0 + f < a.N ? code_value(w[(size_t)(n0 + f) * ld + b * kBlk + k0 + k]) : 0.f;
      }
      __syncthreads();
      for (int k = 0; k < 32; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(xs[2 * tm + i][k0 + k], ws[tn + 16 * j][k], part[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = m0 + 2 * tm + i, f = n0 + tn + 16 * j;
        if (r < rows && f < a.N)
          total[i][j] = fmaf(part[i][j], a.x_scales[(size_t)b * a.lds + source(r)] * w_scales[(size_t)bs_scale_row(f, a.pairs) * a.runs + b], total[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = m0 + 2 * tm + i;
      out[2 * tm + i][tn + 16 * j] = r < rows && a.ep.row_scale ? total[i][j] * a.ep.row_scale[a.order[first + r]] : total[i][j];
    }
  __syncthreads();
  const bool gated = moe_act_gated(a.ep.act);
  const int cols = gated ? TN / 2 : TN, n_out = gated ? a.N / 2 : a.N, c0 = gated ? n0 / 2 : n0;
  for (int i = threadIdx.x; i < TM * cols; i += 256) {
    const int r = i / cols, c = i % cols;
    if (m0 + r >= rows || c0 + c >= n_out) continue;
    const float v = gated ? moe_gated(out[r][2 * c], out[r][2 * c + 1], a.ep.act, a.ep.limit, a.ep.alpha) : moe_act(out[r][c], a.ep.act);
    y[(size_t)(first + m0 + r) * ldy + c0 + c] = from_f32<TO>(v);
  }
}

}  // namespace tib

using namespace tib;

// x: rows [rows, K] in x_dtype (row stride ldx); codes: [rows, ldc], ldc = K rounded up to 128, behind column K zeros; scales:
// [runs of 128 columns, lds], lds at least rows.
TIB_API int tib_quantize_rows(const void* x, int x_dtype, int64_t ldx, void* codes, int64_t ldc, float* scales, int64_t lds, int rows,
                              int K, cudaStream_t stream) {
  if (rows == 0) return TIB_OK;
  if (!x || !codes || !scales || rows < 0 || K < 1) return TIB_E_ARG;
  if (x_dtype != TIB_BF16 && x_dtype != TIB_F32) return TIB_E_DTYPE;
  const int runs = ceil_div(K, kBlk);
  if (ldc < (int64_t)runs * kBlk || lds < rows) return TIB_E_SIZE;
  if (((uintptr_t)codes & 15) || ldc % 16) return TIB_E_ALIGN;
  const int64_t grid = (int64_t)ceil_div(runs, 4) * ceil_div64(rows, 8);
  if (grid > 0x7fffffff) return TIB_E_SIZE;
  const bool vec = ((uintptr_t)x & 15) == 0 && (ldx * (x_dtype == TIB_BF16 ? 2 : 4)) % 16 == 0;
#define TIB_QUANT_GO(T, VEC) \
  TIB_LAUNCH_DEPENDENT((quantize_rows_kernel<T, VEC>), (unsigned)grid, 256, 0, stream, (const T*)x, ldx, (uint8_t*)codes, ldc, scales, lds, rows, K, runs)
  if (x_dtype == TIB_BF16) {
    if (vec) TIB_QUANT_GO(__nv_bfloat16, true);
    else TIB_QUANT_GO(__nv_bfloat16, false);
  } else {
    if (vec) TIB_QUANT_GO(float, true);
    else TIB_QUANT_GO(float, false);
  }
#undef TIB_QUANT_GO
  return TIB_OK;
}

// x: codes [rows, runs * 128] and scales [runs, lds] as tib_quantize_rows leaves them; w: codes [experts, N, runs * 128] and scales
// [experts, scale_rows, runs] (`pairs`: of (gate, up) row pairs); y: [M, N] in y_dtype (row stride ldy), or [M, N / 2] of a gated activation.
// offsets [experts + 1] and order [M]: rows sorted by expert as tib_moe_expert_product takes them; offsets null: one matrix for all rows.
TIB_API int tib_block_scaled_product(const void* x, const float* x_scales, int64_t lds, const void* w, const float* w_scales, int scale_rows,
                                     int pairs, void* y, int y_dtype, int64_t ldy, int M, int N, int runs, const int* offsets,
                                     const int* order, int experts, int top, int x_by_pair, int act, float limit, float alpha,
                                     const float* row_scale, int* error_word, cudaStream_t stream) {
  if (M == 0 || N == 0) return TIB_OK;
  if (!x || !x_scales || !w || !w_scales || !y || M < 0 || N < 0 || runs < 1 || (offsets && (!order || top < 1 || experts < 1))) return TIB_E_ARG;
  if (act < MOE_ACT_NONE || act > MOE_ACT_GELU || (moe_act_gated(act) && (N % 2 || !pairs))) return TIB_E_SIZE;
  if (y_dtype != TIB_BF16 && y_dtype != TIB_F32) return TIB_E_DTYPE;
  BsProduct a;
  a.x = (const uint8_t*)x; a.x_scales = x_scales; a.lds = lds; a.w = (const uint8_t*)w; a.w_scales = w_scales; a.scale_rows = scale_rows;
  a.pairs = pairs; a.M = M; a.N = N; a.runs = runs; a.offsets = offsets; a.order = order; a.experts = experts; a.top = top; a.x_by_pair = x_by_pair;
  a.ep.act = act; a.ep.limit = limit; a.ep.alpha = alpha; a.ep.row_scale = row_scale;
  const int row_tiles = ceil_div(M, 32) + (offsets ? experts : 0);
  if (row_tiles > 65535) return TIB_E_SIZE;
  const dim3 grid(ceil_div(N, 64), row_tiles);
  if (y_dtype == TIB_BF16) TIB_LAUNCH_DEPENDENT((block_scaled_product_kernel<__nv_bfloat16>), grid, 256, 0, stream, a, (__nv_bfloat16*)y, ldy);
  else TIB_LAUNCH_DEPENDENT((block_scaled_product_kernel<float>), grid, 256, 0, stream, a, (float*)y, ldy);
  return TIB_OK;
}

// The calls the Python parts make (common.cuh).
TIB_PACKED(tib_quantize_rows)
TIB_PACKED(tib_block_scaled_product)
