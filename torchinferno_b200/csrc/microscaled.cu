// Rows of activations to 4-bit codes with their scales (microscaled.cuh) and back, and the way of a product with 4-bit matrices to its kernel.
#include "microscaled.cuh"

namespace tib {

// the largest of a block's values, for up to 1024 threads; `scratch`: 32 words, not in use by an earlier call
__device__ __forceinline__ uint32_t ms_block_max(uint32_t v, uint32_t* scratch) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (blockDim.x <= 32) return v;
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  return __reduce_max_sync(0xffffffffu, lane < warps ? scratch[lane] : 0u);
}

// A block takes a row, a thread runs of 16 columns of it, HELD of which it keeps: the row's largest number has to be known before the first code is.  (Wider rows
// are read again, from the L2.)  What is held decides how many blocks an SM has, and these what is on its way.
// What bounds it: its instructions (74 % of the issue slots are used) and memory alike: 8,192 x 14,336 bf16 55 us, 5.4 TB/s; 8,192 x 4,096 17.7 us, in 32 bits 25.8.  (Tried: blocks
// that stay and ask for their next row ahead of this one's codes, 86 and 28 us, of half as many threads an SM.)
template <typename T, bool VEC, int HELD>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? (HELD == 1 ? 5 : HELD == 2 ? 4 : 2) : HELD == 1 ? 6 : HELD == 2 ? 5 : 4)
microscaled_rows_kernel(const T* __restrict__ x, int64_t ldx, int x_rows, unsigned char* __restrict__ codes, unsigned char* __restrict__ scales,
                        float* __restrict__ factors, int rows, int K, int steps, int groups, const int* __restrict__ offsets, const int* __restrict__ order,
                        int experts, int top, int x_by_pair) {
  pdl_trigger();      // (a product behind this kernel asks for its weights while the kernel before is still at work)
  pdl_wait();
  __shared__ uint32_t scratch[32];
  const int row = blockIdx.x, runs = steps * (kMsStep / kMsRun);
  int from = row, tile = row >> 7, group = row >> 3, at = row;      // (at: from the first row of the expert)
  if (offsets) {
    if (row >= bs_offset(offsets, experts, rows)) return;
    int lo = 0, hi = experts;      // offsets[lo] <= row < offsets[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (bs_offset(offsets, mid, rows) <= row) lo = mid; else hi = mid;
    }
    const int first = bs_offset(offsets, lo, rows);
    if (row < first) return;       // (rows ahead of the first expert's are none's)
    at = row - first;
    tile = ms_first_tile(first, lo) + (at >> 7);
    group = ms_first_group(first, lo) + (at >> 3);
    if (x_by_pair) from = min(bs_pair(order, row, rows) / top, x_rows - 1);
  }
  const T* src = x + (size_t)from * ldx;
  uint4 held[HELD][sizeof(T)];
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int run = threadIdx.x + i * blockDim.x;
    bs_ask16<T, VEC>(src + run * kMsRun, run < runs ? K - run * kMsRun : 0, held[i]);
  }
  uint32_t run_largest[HELD];
#pragma unroll
  for (int i = 0; i < HELD; ++i) largest = max(largest, run_largest[i] = bs_largest16<T>(held[i]));
  for (int run = threadIdx.x + HELD * blockDim.x; run < runs; run += blockDim.x) {
    uint4 raw[sizeof(T)];
    bs_ask16<T, VEC>(src + run * kMsRun, K - run * kMsRun, raw);
    largest = max(largest, bs_largest16<T>(raw));
  }
  float r, inverse;
  ms_row_scale(ms_block_max(largest, scratch), r, inverse);
  if (threadIdx.x == 0) factors[row] = r;
  unsigned char* codes_row = codes + (size_t)group * kMsGroupBytes;
  unsigned char* scales_row = scales + (size_t)tile * steps * kMsStepScales + ms_scale_at(at & 127);
  auto finish = [&](int run, const uint4 (&raw)[sizeof(T)], uint32_t run_largest) {      // (whole quarters of a warp: runs and block sizes are multiples of 16)
    if (run >= runs) return;
    uint32_t scale;
    const uint2 c = ms_run_codes<T>(raw, run_largest, inverse, scale);
    *reinterpret_cast<uint2*>(codes_row + (size_t)(run >> 4) * groups * kMsGroupBytes + ms_code_at(at & 7, (run & 15) * (kMsRun / 2))) = c;
    const uint32_t mask = 0xfu << (threadIdx.x & 28), base = threadIdx.x & 28;
    uint32_t four = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) four |= __shfl_sync(mask, scale, base + j) << (8 * j);
    if ((threadIdx.x & 3) == 0) *reinterpret_cast<uint32_t*>(scales_row + (size_t)(run >> 2) * kMsChunkBytes) = four;
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i) finish(threadIdx.x + i * blockDim.x, held[i], run_largest[i]);
  for (int run = threadIdx.x + HELD * blockDim.x; run < runs; run += blockDim.x) {
    uint4 raw[sizeof(T)];
    bs_ask16<T, VEC>(src + run * kMsRun, K - run * kMsRun, raw);
    finish(run, raw, bs_largest16<T>(raw));
  }
}

// The numbers that quantised rows stand for: a thread takes a run.  (s r, four bits and at least 2^-135, is exact.)  8,192 x 14,336: 55 us, 5.5 TB/s; half a run a thread takes
// 72 us, two runs 57.
template <typename TO>
__global__ void __launch_bounds__(256)
microscaled_widen_kernel(MsRows x, TO* __restrict__ out, int64_t ldo, int K, int steps, int per_row, int wide) {
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x / per_row, run = (blockIdx.x - row * per_row) * blockDim.x + threadIdx.x;
  if (run * kMsRun >= K) return;
  const uint2 c = *reinterpret_cast<const uint2*>(x.codes + ((size_t)(run >> 4) * x.groups + (row >> 3)) * kMsGroupBytes + ms_code_at(row & 7, (run & 15) * (kMsRun / 2)));
  const float factor = ms_scale_value(x.scales[((size_t)(row >> 7) * steps * 4 + (run >> 2)) * kMsChunkBytes + ms_scale_at(row & 127) + (run & 3)]) * x.factors[row];
  float v[16];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 p = ms_numbers2(((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 0xffu);
    v[2 * j] = p.x * factor;
    v[2 * j + 1] = p.y * factor;
  }
  TO* dst = out + (size_t)row * ldo + run * kMsRun;
  TO w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = from_f32<TO>(v[j]);
  if (wide && run * kMsRun + kMsRun <= K) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(TO); ++j) reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(w)[j];
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (run * kMsRun + j < K) dst[j] = w[j];
  }
}

}  // namespace tib

using namespace tib;

// x: rows [x_rows, K] in x_dtype (row stride ldx); codes, scales, factors: as microscaled.cuh has them, of `rows` rows.  offsets [experts + 1] (and with x_by_pair order
// [rows]: row m is made of row order[m] / top of x, else of row m): rows sorted by expert; null: one matrix for all.
TIB_API int tib_microscaled_rows(const void* x, int x_dtype, int64_t ldx, int x_rows, void* codes, void* scales, float* factors, int rows, int K,
                                 const int* offsets, const int* order, int experts, int top, int x_by_pair, cudaStream_t stream) {
  if (rows == 0) return TIB_OK;
  if (!x || !codes || !scales || !factors || rows < 0 || K < 1 || x_rows < 1 || experts < 1 || top < 1) return TIB_E_ARG;
  if ((offsets && x_by_pair) ? !order : x_rows < rows) return TIB_E_ARG;
  if (x_dtype != TIB_BF16 && x_dtype != TIB_F32) return TIB_E_DTYPE;
  if (((uintptr_t)codes | (uintptr_t)scales) & 15) return TIB_E_ALIGN;
  // (Of many rows twice as many runs a thread: twice as many rows at a time on an SM.  8,192 rows of 4,096 21.4 us with one, 17.9 with two.)
  const int steps = ms_steps(K), runs = steps * (kMsStep / kMsRun), held = runs <= (rows > 592 ? 128 : 256) ? 1 : runs <= (rows > 592 ? 256 : 512) ? 2 : 4;
  const int threads = runs >= 256 * held ? 256 : (ceil_div(runs, held) + 31) / 32 * 32;
  const bool vec = ((uintptr_t)x & 15) == 0 && (ldx * (x_dtype == TIB_BF16 ? 2 : 4)) % 16 == 0;
#define TIB_MS_ROWS_HELD(T, VEC, HELD)                                                                                                                      \
  TIB_LAUNCH_DEPENDENT((microscaled_rows_kernel<T, VEC, HELD>), (unsigned)rows, threads, 0, stream, (const T*)x, ldx, x_rows, (unsigned char*)codes,          \
                       (unsigned char*)scales, factors, rows, K, steps, ms_groups(rows, offsets ? experts : 0), offsets, order, experts, top, x_by_pair)
#define TIB_MS_ROWS_GO(T, VEC)                        \
  do {                                                \
    if (held == 1) TIB_MS_ROWS_HELD(T, VEC, 1);       \
    else if (held == 2) TIB_MS_ROWS_HELD(T, VEC, 2);  \
    else TIB_MS_ROWS_HELD(T, VEC, 4);                 \
  } while (0)
  if (x_dtype == TIB_BF16) {
    if (vec) TIB_MS_ROWS_GO(__nv_bfloat16, true);
    else TIB_MS_ROWS_GO(__nv_bfloat16, false);
  } else {
    if (vec) TIB_MS_ROWS_GO(float, true);
    else TIB_MS_ROWS_GO(float, false);
  }
#undef TIB_MS_ROWS_GO
#undef TIB_MS_ROWS_HELD
  return TIB_OK;
}

// The numbers [rows, K] that rows as tib_microscaled_rows leaves them (offsets null) stand for, in out_dtype (row stride ldo).
TIB_API int tib_microscaled_widen(const void* codes, const void* scales, const float* factors, void* out, int out_dtype, int64_t ldo, int rows, int K,
                                  cudaStream_t stream) {
  if (rows == 0) return TIB_OK;
  if (!codes || !scales || !factors || !out || rows < 0 || K < 1) return TIB_E_ARG;
  if (out_dtype != TIB_BF16 && out_dtype != TIB_F32) return TIB_E_DTYPE;
  if (((uintptr_t)codes | (uintptr_t)scales) & 15) return TIB_E_ALIGN;
  const int runs = ceil_div(K, kMsRun), threads = runs >= 256 ? 256 : (runs + 31) / 32 * 32, per_row = ceil_div(runs, threads);
  const int64_t grid = (int64_t)rows * per_row;
  if (grid > 0x7fffffff) return TIB_E_SIZE;
  const MsRows r{(const unsigned char*)codes, (const unsigned char*)scales, factors, ms_groups(rows, 0)};
  const int wide = ((uintptr_t)out & 15) == 0 && (ldo * (out_dtype == TIB_BF16 ? 2 : 4)) % 16 == 0;
  if (out_dtype == TIB_BF16) TIB_LAUNCH_DEPENDENT(microscaled_widen_kernel<__nv_bfloat16>, (unsigned)grid, threads, 0, stream, r, (__nv_bfloat16*)out, ldo, K, ms_steps(K), per_row, wide);
  else TIB_LAUNCH_DEPENDENT(microscaled_widen_kernel<float>, (unsigned)grid, threads, 0, stream, r, (float*)out, ldo, K, ms_steps(K), per_row, wide);
  return TIB_OK;
}

// A product as its callers see it: y [M, N] (or [M, N / 2] of a gated activation) in y_dtype, row stride ldy.  codes, scales, factors: where the quantised rows
// are, or (`make`) are put first, from rows x [x_rows, K].  w: codes, scales and factors [experts, N] of the matrices (`pairs`: 1 of (gate, up) row pairs; 2 more where a factor that
// matters is outside 2^-100 .. 2^70: these run on pairs of SMs).
// offsets [experts + 1], order [M], top, x_by_pair: rows sorted by expert as tib_moe_expert_product takes them; offsets null: one matrix for all rows.
TIB_API int tib_microscaled_product(const void* w, const void* w_scales, const float* w_factors, int pairs, int N, int K, int experts, const void* x, int x_dtype,
                                    int64_t ldx, int x_rows, void* codes, void* scales, float* factors, int make, void* y, int y_dtype, int64_t ldy, int M,
                                    const int* offsets, const int* order, int top, int x_by_pair, int act, float limit, float alpha, const float* row_scale,
                                    int* error_word, cudaStream_t stream) {
  if (M == 0 || N == 0) return TIB_OK;
  const bool made_inside = make && !codes;
  if ((!made_inside && (!codes || !scales || !factors)) || !w || !w_scales || !w_factors || !y || M < 0 || N < 0 || K < 1 || experts < 1 || top < 1) return TIB_E_ARG;
  if ((offsets && !order) || (row_scale && !order)) return TIB_E_ARG;
  if (act < MOE_ACT_NONE || act > MOE_ACT_GELU || (moe_act_gated(act) && !(pairs & 1)) || ((pairs & 1) && N % 2)) return TIB_E_SIZE;
  const bool far = pairs & 2;
  if (y_dtype != TIB_BF16 && y_dtype != TIB_F32) return TIB_E_DTYPE;
  if (((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)w | (uintptr_t)w_scales) & 15) return TIB_E_ALIGN;
  if (made_inside) {      // (every block reads the rows while others write y)
    if (!x || offsets || far || M > x_rows || !ms_makes_rows(M, N, K)) return TIB_E_ARG;
    if (x_dtype != TIB_BF16) return TIB_E_DTYPE;
    if (((uintptr_t)x & 15) || ldx % 8) return TIB_E_ALIGN;
    const char *from = (const char*)x, *to = (const char*)y;
    const int width = moe_act_gated(act) ? N / 2 : N;
    if (from < to + ((int64_t)(M - 1) * ldy + width) * (y_dtype == TIB_BF16 ? 2 : 4) && to < from + ((int64_t)(M - 1) * ldx + K) * 2) return TIB_E_ARG;
  } else if (make) {
    const int rc = tib_microscaled_rows(x, x_dtype, ldx, x_rows, codes, scales, factors, M, K, offsets, order, experts, top, x_by_pair, stream);
    if (rc != TIB_OK) return rc;
  }
  MsArgs a;
  a.x = MsRows{(const unsigned char*)codes, (const unsigned char*)scales, factors, ms_groups(M, offsets ? experts : 0)};
  a.w = (const unsigned char*)w; a.w_scales = (const unsigned char*)w_scales; a.w_factors = w_factors;
  a.M = M; a.N = N; a.steps = ms_steps(K); a.stages = a.tmem_cols = 0; a.offsets = offsets; a.order = order; a.experts = experts;
  a.limit = limit; a.alpha = alpha; a.row_scale = row_scale; a.error_word = error_word;
  a.made = made_inside ? (const __nv_bfloat16*)x : nullptr; a.ld_made = ldx; a.K = K;
  if (!made_inside && (far || ms_on_pairs_of_sms(M, N, a.steps, offsets ? experts : 0))) return ms_product_2cta(a, act, y, y_dtype, ldy, stream);
  return ms_product_tcgen05(a, act, y, y_dtype, ldy, stream);
}

// How a product of M rows with one matrix (experts 0) or sorted by expert runs where its factors are ordinary: {rows of a tile at most (256: on pairs of SMs), blocks that share a tile, steps of a block at
// most, stages of its ring}.
TIB_API int tib_microscaled_plan(int M, int N, int K, int experts, int* plan) {
  if (!plan || M < 1 || N < 1 || K < 1 || experts < 0) return TIB_E_ARG;
  const int steps = ms_steps(K);
  return ms_on_pairs_of_sms(M, N, steps, experts) ? ms_plan_2cta(M, N, steps, experts, plan) : ms_plan_tcgen05(M, N, steps, experts, plan);
}

// What a block of such a product takes of an SM: {columns of tensor memory (of 512), bytes of shared memory} (smem_for_tmem).
TIB_API int tib_microscaled_room(int M, int N, int K, int experts, int* room) {
  if (!room || M < 1 || N < 1 || K < 1 || experts < 0) return TIB_E_ARG;
  return ms_on_pairs_of_sms(M, N, ms_steps(K), experts) ? ms_room_2cta(experts, room) : ms_room_tcgen05(M, N, ms_steps(K), experts, room);
}

// Whether tib_microscaled_product makes the codes of M rows of 16-bit numbers (16-byte aligned, as is a row's stride) for one matrix without room for them (codes null).
TIB_API int tib_microscaled_makes(int M, int N, int K, int* answer) {
  if (!answer || M < 1 || N < 1 || K < 1) return TIB_E_ARG;
  *answer = ms_makes_rows(M, N, K);
  return TIB_OK;
}

TIB_PACKED(tib_microscaled_rows)
TIB_PACKED(tib_microscaled_makes)
TIB_PACKED(tib_microscaled_widen)
TIB_PACKED(tib_microscaled_product)
TIB_PACKED(tib_microscaled_plan)
TIB_PACKED(tib_microscaled_room)
