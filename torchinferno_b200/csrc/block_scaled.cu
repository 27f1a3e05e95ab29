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
                     int64_t lds, int rows, int K, int runs, const int* __restrict__ order, int top, const int* __restrict__ sorted) {
  pdl_wait();
  pdl_trigger();
  // thread = (row of 8, run of 4, eighth of the run)
  const int groups = (runs + 3) >> 2, row8 = blockIdx.x / groups;
  const int eighth = threadIdx.x & 7, row = row8 * 8 + (threadIdx.x >> 5), run = (blockIdx.x - row8 * groups) * 4 + ((threadIdx.x >> 3) & 3);
  const bool in = row < (order ? min(rows, *sorted) : rows) && run < runs;
  const int col = run * kBlk + eighth * 16, from = !in ? 0 : order ? order[row] / top : row;
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

// x: rows [rows, K] in x_dtype (row stride ldx); codes: [rows, ldc], ldc = K rounded up to 128, behind column K zeros; scales:
// [runs of 128 columns, lds], lds at least rows.  order [rows]: row r is made of row order[r] / top of x, for the first *sorted rows; null: of row r.
TIB_API int tib_quantize_rows(const void* x, int x_dtype, int64_t ldx, void* codes, int64_t ldc, float* scales, int64_t lds, int rows,
                              int K, const int* order, int top, const int* sorted, cudaStream_t stream) {
  if (rows == 0) return TIB_OK;
  if (!x || !codes || !scales || rows < 0 || K < 1 || (order && (top < 1 || !sorted))) return TIB_E_ARG;
  if (x_dtype != TIB_BF16 && x_dtype != TIB_F32) return TIB_E_DTYPE;
  const int runs = ceil_div(K, kBlk);
  if (ldc < (int64_t)runs * kBlk || lds < rows) return TIB_E_SIZE;
  if (((uintptr_t)codes & 15) || ldc % 16) return TIB_E_ALIGN;
  const int64_t grid = (int64_t)ceil_div(runs, 4) * ceil_div64(rows, 8);
  if (grid > 0x7fffffff) return TIB_E_SIZE;
  const bool vec = ((uintptr_t)x & 15) == 0 && (ldx * (x_dtype == TIB_BF16 ? 2 : 4)) % 16 == 0;
#define TIB_QUANT_GO(T, VEC) \
  TIB_LAUNCH_DEPENDENT((quantize_rows_kernel<T, VEC>), (unsigned)grid, 256, 0, stream, (const T*)x, ldx, (uint8_t*)codes, ldc, scales, lds, rows, K, runs, order, top, sorted)
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

// The calls the Python parts make (common.cuh).
TIB_PACKED(tib_quantize_rows)
