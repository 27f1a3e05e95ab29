// Rows of activations to 8-bit codes with a power of two for each run of 128 columns (block_scaled.cuh).
//
// Eight lanes take a run, 16 columns each: their largest absolute value by its bits as an integer (a NaN is then the
// largest of all, where a maximum of floats would pass over it), a butterfly of three steps, one multiplication and one
// conversion a number.  A block takes eight rows and four runs of each, so that the scales of a run, which lie row after row, are written 32 bytes
// at a time.  What bounds it: memory (8,192 x 14,336 bf16: 57.9 us, 94 % of the measured copy bandwidth).
#include "block_scaled.cuh"

namespace tib {

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scales,
                     int64_t lds, int rows, int K, int runs, const int* __restrict__ order, int top, const int* __restrict__ sorted, int x_rows) {
  pdl_wait();
  pdl_trigger();
  // thread = (row of 8, run of 4, eighth of the run)
  const int groups = (runs + 3) >> 2, row8 = blockIdx.x / groups;
  const int eighth = threadIdx.x & 7, row = row8 * 8 + (threadIdx.x >> 5), run = (blockIdx.x - row8 * groups) * 4 + ((threadIdx.x >> 3) & 3);
  const bool in = row < (order ? min(rows, *sorted) : rows) && run < runs;
  const int col = run * kBlk + eighth * 16, from = !in ? 0 : order ? min(bs_pair(order, row, rows) / top, x_rows - 1) : row;
  uint4 raw[sizeof(T)];
  bs_ask16<T, VEC>(x + (size_t)from * ldx + (in ? col : 0), in ? K - col : 0, raw);
  uint32_t largest = bs_largest16<T>(raw);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  float scale, inverse;
  bs_run_scale(largest, scale, inverse);
  if (!in) return;
  *reinterpret_cast<uint4*>(codes + (size_t)row * ldc + col) = bs_codes16<T>(raw, inverse);
  if (eighth == 0) scales[(size_t)run * lds + row] = scale;
}

}  // namespace tib

using namespace tib;

// x: rows [x_rows, K] in x_dtype (row stride ldx); codes: [rows, ldc], ldc = K rounded up to 128, behind column K zeros; scales:
// [runs of 128 columns, lds], lds at least rows.  order [rows]: row r is made of row order[r] / top of x, for the first *sorted rows; null: of row r.
TIB_API int tib_quantize_rows(const void* x, int x_dtype, int64_t ldx, void* codes, int64_t ldc, float* scales, int64_t lds, int rows,
                              int K, const int* order, int top, const int* sorted, int x_rows, cudaStream_t stream) {
  if (rows == 0) return TIB_OK;
  if (!x || !codes || !scales || rows < 0 || K < 1 || (order ? top < 1 || !sorted || x_rows < 1 : x_rows < rows)) return TIB_E_ARG;
  if (x_dtype != TIB_BF16 && x_dtype != TIB_F32) return TIB_E_DTYPE;
  const int runs = ceil_div(K, kBlk);
  if (ldc < (int64_t)runs * kBlk || lds < rows) return TIB_E_SIZE;
  if (((uintptr_t)codes & 15) || ldc % 16) return TIB_E_ALIGN;
  const int64_t grid = (int64_t)ceil_div(runs, 4) * ceil_div64(rows, 8);
  if (grid > 0x7fffffff) return TIB_E_SIZE;
  const bool vec = ((uintptr_t)x & 15) == 0 && (ldx * (x_dtype == TIB_BF16 ? 2 : 4)) % 16 == 0;
#define TIB_QUANT_GO(T, VEC) \
  TIB_LAUNCH_DEPENDENT((quantize_rows_kernel<T, VEC>), (unsigned)grid, 256, 0, stream, (const T*)x, ldx, (uint8_t*)codes, ldc, scales, lds, rows, K, runs, order, top, sorted, x_rows)
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

// Whether a product of codes runs on pairs of SMs, in tiles of 256 rows x 256 features: where tiles of 128 x 128 would be more than one for each of 148 SMs.
// (us, tiles of 128 / pairs: 4,096 -> 4,096 512 rows 22.9 / 22.8, 768 rows 39 / 24; 4,096 -> 6,144 384 rows 23.1 / 25.2, 512 rows 39 / 26; 14,336 -> 4,096
// 512 rows 62 / 60, 768 rows 110 / 62.)  Up to 128 rows the weights are the work: 4,096 -> 28,672 128 rows 38 / 42, 64 rows 29 / 39, 192 rows 69 / 42.
static bool on_pairs_of_sms(int rows, int features) { return rows > 128 && (int64_t)ceil_div(rows, 128) * ceil_div(features, 128) > 148; }

// Rows sorted by expert run there from so many rows an expert on, on average.  (32 experts 2,048 -> 1,024, us, tiles of 128 / pairs: 64 rows an expert 26.2 / 27.6,
// 96 28.2 / 29.2, 128 37.2 / 29.8, 192 47.8 / 32.6, 256 60.7 / 45.1, 512 98.4 / 71.4; gated, 256: 95.3 / 73.9.)
constexpr int kBsPairRows = 100;

static bool takes_pairs_of_sms(int M, int N, int experts) {      // experts: 0 for one matrix
  return experts ? M >= (int64_t)experts * kBsPairRows && experts <= tib_block_scaled_2cta_experts() : on_pairs_of_sms(M, N);
}

// How a product runs whose rows come as they are (codes 0) or as codes: {rows of a tile at most, blocks that share a tile, steps of a block at most, stages of its
// ring}; tiles of 256 rows are those of pairs of SMs.  experts: 0 for one matrix.
TIB_API int tib_block_scaled_plan(int codes, int M, int N, int K, int experts, int* plan) {
  if (!codes || !takes_pairs_of_sms(M, N, experts)) return tib_block_scaled_tcgen05_plan(codes, M, N, K, experts, plan);
  return tib_block_scaled_2cta_plan(M, N, K, experts, plan);
}

// A product as its callers see it: rows x [x_rows, K] times matrices in blocks (the other arguments as tib_block_scaled_tcgen05).  codes: where the rows'
// codes [M, runs * 128] and scales [runs, M rounded up to 4] go, ahead of the product (`make`; not made: they are there from a call before); null: the
// product's kernel quantises the rows itself.
TIB_API int tib_block_scaled_product(const void* x, int x_dtype, int64_t ldx, int x_rows, void* codes, int make, const void* w, const float* w_scales,
                                     int scale_rows, int pairs, void* y, int y_dtype, int64_t ldy, int M, int N, int K, const int* offsets,
                                     const int* order, int experts, int top, int x_by_pair, int act, float limit, float alpha,
                                     const float* row_scale, float far_low, float far_high, int* error_word, cudaStream_t stream) {
  if (M == 0 || N == 0) return TIB_OK;
  if (!codes)
    return tib_block_scaled_tcgen05(x, x_dtype, ldx, x_rows, nullptr, 0, w, w_scales, scale_rows, pairs, y, y_dtype, ldy, M, N, K, offsets, order, experts,
                                    top, x_by_pair, act, limit, alpha, row_scale, far_low, far_high, error_word, stream);
  if (M < 0 || K < 1 || (offsets && experts < 1)) return TIB_E_ARG;
  const int runs = ceil_div(K, kBlk);
  const int64_t lds = ((int64_t)M + 3) & ~(int64_t)3;
  float* scales = reinterpret_cast<float*>(static_cast<char*>(codes) + (int64_t)M * runs * kBlk);
  if (make) {
    const bool gather = offsets && x_by_pair;      // (the pairs' rows, sorted on the way)
    const int rc = tib_quantize_rows(x, x_dtype, ldx, codes, (int64_t)runs * kBlk, scales, lds, M, K, gather ? order : nullptr, top,
                                     gather ? offsets + experts : nullptr, x_rows, stream);
    if (rc != TIB_OK) return rc;
  }
  if (takes_pairs_of_sms(M, N, offsets ? experts : 0))
    return tib_block_scaled_2cta(codes, scales, lds, w, w_scales, scale_rows, pairs, y, y_dtype, ldy, M, N, K, offsets, order, experts, act, limit, alpha,
                                 row_scale, far_low, far_high, error_word, stream);
  return tib_block_scaled_tcgen05(codes, -1, 0, M, scales, lds, w, w_scales, scale_rows, pairs, y, y_dtype, ldy, M, N, K, offsets, order, experts, top, 0, act,
                                  limit, alpha, row_scale, far_low, far_high, error_word, stream);
}

// The calls the Python parts make (common.cuh).
TIB_PACKED(tib_quantize_rows)
TIB_PACKED(tib_block_scaled_product)
TIB_PACKED(tib_block_scaled_plan)
