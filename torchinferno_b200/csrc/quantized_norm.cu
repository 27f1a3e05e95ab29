// Root-mean-square norm with the residual's addition, as tib_add_rmsnorm, whose rows leave as codes and scales: in 4 bits (microscaled.cuh) or in 8
// (block_scaled.cuh).
//     h = residual + delta (32 bits; kept as the next residual),  v = h / sqrt(mean(h^2) + eps) * weight, rounded to the rows' type,  codes and scales of v
// A block takes a row.  The sums run in tib_add_rmsnorm's order and the codes are made of what it writes, so that codes, scales and residual are bit for
// bit those of the three steps one by one.
// It lets the kernel behind it in before it waits for the one ahead.  That is as good for whoever waits: a kernel is over only when the one ahead of it is.  (What kernels
// behind it may read before they wait: see launch_dependent.)
// What bounds it: memory.  8,192 x 4,096 bf16: 61.7 us for 354 MB (5.7 TB/s; tib_add_rmsnorm, whose rows leave in bf16, takes 60.9, and codes made behind it 17.7 more), in 32 bits
// 69 us for 421 MB; eight rows 2.9 us, where tib_add_rmsnorm takes 2.5 and the codes 2.
#include "microscaled.cuh"

namespace tib {

constexpr int kQnHeld = 8, kQnWidth = 8 * 1024;      // columns of a thread of those that norm a row, of a row that a block keeps
constexpr int kQnFoursWidth = 16 * 1024;             // the same of a row read four columns a load

struct QnArgs {
  const void* delta;           // [rows, hidden] in the rows' type, or null
  const float* residual;
  float* sum;                  // where h goes: null where it is not kept
  const int* rows;             // or null: every row
  const float* weight;
  void* out;                   // the normed rows [n_out, hidden], or null
  unsigned char* codes;        // 4 bits: [steps, groups, 1024]; 8 bits: [n_out, runs * 128]
  unsigned char* scales;       // of 4 bits
  float* factors;              // 4 bits: [n_out]; 8 bits: the scales [runs, lds]
  int64_t lds;
  int hidden;
  float eps;
  int groups, n_rows;          // n_rows: of the residual
};

// The row of the residual that row `orow` is (an index is kept within what there is)
__device__ __forceinline__ int qn_row(const QnArgs& a, int orow) { return a.rows ? min(max(a.rows[orow], 0), a.n_rows - 1) : orow; }

// Eight numbers to eight 8-bit codes
__device__ __forceinline__ uint2 qn_bytes8(const float (&v)[8], float inverse) {
  return make_uint2(bs_codes4(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse),
                    bs_codes4(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse));
}
template <typename T> __device__ __forceinline__ uint32_t qn_largest8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// block_sum (common.cuh), bit for bit, with one barrier: every warp adds up the warps' sums as the first does there.  `scratch` (32 floats) is not in use by an earlier call.
__device__ __forceinline__ float qn_block_sum(float v, float* scratch) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum(lane < (int)((blockDim.x + 31) >> 5) ? scratch[lane] : 0.f);
}

// What a thread does with eight numbers of a row (columns 8 g .. of it, zeros behind the last); all threads of a warp call it together.  largest: of the row
// (4 bits).  Two threads have a run of 16, sixteen one of 128.
template <typename T, bool BYTES>
__device__ __forceinline__ void qn_codes8(const QnArgs& a, int row, int g, const float (&v)[8], float r, float inverse, int steps) {
  uint32_t m = qn_largest8<T>(v);
  if constexpr (BYTES) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int runs = (a.hidden + kBlk - 1) / kBlk;
    float s, back;
    bs_run_scale(m, s, back);
    if (g < runs * 16) *reinterpret_cast<uint2*>(a.codes + (size_t)row * runs * kBlk + g * 8) = qn_bytes8(v, back);
    if (g < runs * 16 && (g & 15) == 0) a.factors[(size_t)(g >> 4) * a.lds + row] = s;
  } else {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const uint32_t scale = inverse == 0.f ? 0u : ms_run_scale<T>(__uint_as_float(m) * inverse);
    const uint32_t c = scale == 0 ? 0u : ms_codes8<T>(v, inverse, ms_reciprocal(ms_scale_value(scale)));
    uint32_t four = scale << (8 * ((g >> 1) & 3));
    four |= __shfl_xor_sync(0xffffffffu, four, 2);
    four |= __shfl_xor_sync(0xffffffffu, four, 4);
    if (g >= steps * (kMsStep / 8)) return;
    *reinterpret_cast<uint32_t*>(a.codes + ((size_t)(g >> 5) * a.groups + (row >> 3)) * kMsGroupBytes + ms_code_at(row & 7, (g & 31) * 4)) = c;
    if ((g & 7) == 0)
      *reinterpret_cast<uint32_t*>(a.scales + ((size_t)(row >> 7) * steps * 4 + (g >> 3)) * kMsChunkBytes + ms_scale_at(row & 127)) = four;
    if (g == 0) a.factors[row] = r;
  }
}

__device__ __forceinline__ uint32_t qn_block_max(uint32_t v, uint32_t* scratch) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return __reduce_max_sync(0xffffffffu, lane < (int)(blockDim.x >> 5) ? scratch[lane] : 0u);
}

// bf16 rows whose width is a multiple of 8 and at most 8 * 1024: a thread keeps its eight numbers (as add_rmsnorm_bf16x8_kernel does), so the row is
// read once.  The block's threads, a multiple of 32, cover whole steps of 256 columns.  The weight is asked for with the row, not
// behind its sum: with that and the sum's one barrier 8 rows of 2,048 take 1.9 us (before 2.1), 592 of 4,096 6.4 (6.75), 8,192 of them the same within 1 %.
template <bool BYTES>
__global__ void __launch_bounds__(1024)
quantized_norm_bf16x8_kernel(const QnArgs a) {
  pdl_trigger();      // (see microscaled_rows_kernel)
  pdl_wait();
  __shared__ float scratch[32];
  __shared__ uint32_t scratch_max[32];
  const int orow = blockIdx.x, srow = qn_row(a, orow), c = threadIdx.x * 8;
  const bool active = c < a.hidden;
  float h[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float ss = 0.f;
  float4 w0 = make_float4(0.f, 0.f, 0.f, 0.f), w1 = w0;
  if (active) {
    w0 = *reinterpret_cast<const float4*>(a.weight + c);
    w1 = *reinterpret_cast<const float4*>(a.weight + c + 4);
    const size_t at = (size_t)srow * a.hidden + c;
    const float4 r0 = *reinterpret_cast<const float4*>(a.residual + at), r1 = *reinterpret_cast<const float4*>(a.residual + at + 4);
    h[0] = r0.x; h[1] = r0.y; h[2] = r0.z; h[3] = r0.w; h[4] = r1.x; h[5] = r1.y; h[6] = r1.z; h[7] = r1.w;
    if (a.delta) {
      const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.delta) + at);
      const __nv_bfloat162* d2 = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = bf16x2_floats(d2[i]);
        h[2 * i] += f.x;
        h[2 * i + 1] += f.y;
      }
    }
    if (a.sum) {
      *reinterpret_cast<float4*>(a.sum + at) = make_float4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<float4*>(a.sum + at + 4) = make_float4(h[4], h[5], h[6], h[7]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += h[i] * h[i];
  }
  const float total = qn_block_sum(ss, scratch);
  const float inv = rsqrtf(total / (float)a.hidden + a.eps);
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (active) {
    const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    uint4 packed;
    __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o2[i] = __floats2bfloat162_rn(h[2 * i] * inv * w[2 * i], h[2 * i + 1] * inv * w[2 * i + 1]);
      const float2 f = bf16x2_floats(o2[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
    if (a.out) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + (size_t)orow * a.hidden + c) = packed;
  }
  float r = 1.f, inverse = 1.f;
  if constexpr (!BYTES) ms_row_scale(qn_block_max(qn_largest8<__nv_bfloat16>(v), scratch_max), r, inverse);
  qn_codes8<__nv_bfloat16, BYTES>(a, orow, threadIdx.x, v, r, inverse, (a.hidden + kMsStep - 1) / kMsStep);
}

// Four neighbours of a row, in 32 bits and back (rounded: what comes back is what was stored).
__device__ __forceinline__ float4 qn_load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 qn_load4(const __nv_bfloat16* p) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u));
}
__device__ __forceinline__ float4 qn_store4(float* p, float4 v) {
  if (p) *reinterpret_cast<float4*>(p) = v;
  return v;
}
__device__ __forceinline__ float4 qn_store4(__nv_bfloat16* p, float4 v) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
  if (p) *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  return make_float4(__low2float(lo), __high2float(lo), __low2float(hi), __high2float(hi));
}

// Rows of a multiple of four columns, up to 16 * 1024: four columns a load.  The sums are those of `virtuals` threads that each add up every virtuals-th column
// (add_rmsnorm_kernel's), of which a thread is four neighbours: what is a shuffle over 1 and 2 lanes there is an addition here, what is one over 4, 8 and 16 one
// over 1, 2 and 4.  A quarter of the threads a row is four times as many rows on an SM.  Of long rows eight loads a thread are asked for at a time: all 16 ahead of
// the first sum take more registers than two blocks an SM leave (2,048 rows of 16,384 in bf16: 89 us, so 106; quantized_norm_kernel takes 179).
// 8 rows of 14,336 in bf16 take 7.7 us (12.4 there; the norm and the codes by two kernels 9.8).
template <typename T, bool BYTES, int HELD>
__global__ void __launch_bounds__(256, HELD <= 4 ? 5 : HELD <= 8 ? 3 : 2)
quantized_norm_x4_kernel(const QnArgs a, int virtuals) {
  pdl_trigger();      // (see microscaled_rows_kernel)
  pdl_wait();
  extern __shared__ float normed_row[];      // [hidden rounded up to 256]
  __shared__ float scratch[32];
  __shared__ uint32_t scratch_max[32];
  const int orow = blockIdx.x, srow = qn_row(a, orow), lane = threadIdx.x & 31;
  const size_t at = (size_t)srow * a.hidden;
  const T* delta = static_cast<const T*>(a.delta);
  T* out = a.out ? static_cast<T*>(a.out) + (size_t)orow * a.hidden : nullptr;
  const int c0 = threadIdx.x * 4 < virtuals ? threadIdx.x * 4 : a.hidden;      // (threads beyond have no column)
  constexpr int ASKED = HELD < 8 ? HELD : 8;      // (at a time: registers)
  float4 h[HELD], ss = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int first = 0; first < HELD; first += ASKED) {
    float4 d[ASKED];
#pragma unroll
    for (int i = 0; i < ASKED; ++i) {
      const int c = c0 + (first + i) * virtuals;
      h[first + i] = d[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < a.hidden) {
        h[first + i] = qn_load4(a.residual + at + c);
        if (delta) d[i] = qn_load4(delta + at + c);
      }
    }
#pragma unroll
    for (int i = 0; i < ASKED; ++i) {
      const int c = c0 + (first + i) * virtuals;
      float4& v = h[first + i];
      if (c >= a.hidden) break;
      if (delta) v = make_float4(v.x + d[i].x, v.y + d[i].y, v.z + d[i].z, v.w + d[i].w);
      if (a.sum) *reinterpret_cast<float4*>(a.sum + at + c) = v;
      ss.x += v.x * v.x; ss.y += v.y * v.y; ss.z += v.z * v.z; ss.w += v.w * v.w;
    }
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    ss.x += __shfl_xor_sync(0xffffffffu, ss.x, o);
    ss.y += __shfl_xor_sync(0xffffffffu, ss.y, o);
    ss.z += __shfl_xor_sync(0xffffffffu, ss.z, o);
    ss.w += __shfl_xor_sync(0xffffffffu, ss.w, o);
  }
  const float part = (ss.x + ss.z) + (ss.y + ss.w);
  if ((threadIdx.x & 7) == 0 && threadIdx.x * 4 < virtuals) scratch[threadIdx.x >> 3] = part;
  __syncthreads();
  const float total = warp_sum(lane < virtuals >> 5 ? scratch[lane] : 0.f);
  const float inv = rsqrtf(total / (float)a.hidden + a.eps);
  const int steps = (a.hidden + kMsStep - 1) / kMsStep, eights = steps * (kMsStep / 8);
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int c = c0 + i * virtuals;
    if (c >= a.hidden) break;
    const float4 w = *reinterpret_cast<const float4*>(a.weight + c);
    const float4 y = qn_store4(out ? out + c : nullptr, make_float4(h[i].x * inv * w.x, h[i].y * inv * w.y, h[i].z * inv * w.z, h[i].w * inv * w.w));
    *reinterpret_cast<float4*>(normed_row + c) = y;
    largest = max(max(max(largest, __float_as_uint(y.x) & 0x7fffffffu), max(__float_as_uint(y.y) & 0x7fffffffu, __float_as_uint(y.z) & 0x7fffffffu)), __float_as_uint(y.w) & 0x7fffffffu);
  }
  for (int c = a.hidden + threadIdx.x; c < steps * kMsStep; c += blockDim.x) normed_row[c] = 0.f;
  float r = 1.f, inverse = 1.f;
  if constexpr (BYTES) __syncthreads();
  else ms_row_scale(qn_block_max(largest, scratch_max), r, inverse);      // (a barrier of the block)
  for (int g = threadIdx.x; g < eights; g += blockDim.x) {                // (whole warps: both are multiples of 32)
    float v[8];
    const float4 lo = reinterpret_cast<const float4*>(normed_row)[2 * g], hi = reinterpret_cast<const float4*>(normed_row)[2 * g + 1];
    v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    qn_codes8<T, BYTES>(a, orow, g, v, r, inverse, steps);
  }
}

// Any other width up to 8 * 1024, either type: the sums in add_rmsnorm_kernel's order (columns in turn, so many a thread that 8 hold them), the codes eight columns a
// thread: in between the normed row crosses shared memory.
template <typename T, bool BYTES>
__global__ void __launch_bounds__(1024)
quantized_norm_held_kernel(const QnArgs a) {
  pdl_trigger();      // (see microscaled_rows_kernel)
  pdl_wait();
  extern __shared__ float normed_row[];      // [hidden rounded up to 256]
  __shared__ float scratch[32];
  __shared__ uint32_t scratch_max[32];
  const int orow = blockIdx.x, srow = qn_row(a, orow);
  const size_t at = (size_t)srow * a.hidden;
  const T* delta = static_cast<const T*>(a.delta);
  float h[kQnHeld];
#pragma unroll
  for (int i = 0; i < kQnHeld; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    h[i] = c < a.hidden ? a.residual[at + c] : 0.f;
    if (delta && c < a.hidden) h[i] += to_f32(delta[at + c]);
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kQnHeld; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c >= a.hidden) break;
    if (a.sum) a.sum[at + c] = h[i];
    ss += h[i] * h[i];
  }
  const float total = qn_block_sum(ss, scratch);
  const float inv = rsqrtf(total / (float)a.hidden + a.eps);
  const int steps = (a.hidden + kMsStep - 1) / kMsStep, eights = steps * (kMsStep / 8);
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < kQnHeld; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c >= a.hidden) break;
    const T y = from_f32<T>(h[i] * inv * a.weight[c]);
    if (a.out) static_cast<T*>(a.out)[(size_t)orow * a.hidden + c] = y;
    normed_row[c] = to_f32(y);
    largest = max(largest, __float_as_uint(normed_row[c]) & 0x7fffffffu);
  }
  for (int c = a.hidden + threadIdx.x; c < steps * kMsStep; c += blockDim.x) normed_row[c] = 0.f;
  float r = 1.f, inverse = 1.f;
  if constexpr (BYTES) __syncthreads();
  else ms_row_scale(qn_block_max(largest, scratch_max), r, inverse);      // (a barrier of the block)
  for (int g = threadIdx.x; g < eights; g += blockDim.x) {                // (whole warps: both are multiples of 32)
    float v[8];
    const float4 lo = reinterpret_cast<const float4*>(normed_row)[2 * g], hi = reinterpret_cast<const float4*>(normed_row)[2 * g + 1];
    v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    qn_codes8<T, BYTES>(a, orow, g, v, r, inverse, steps);
  }
}

// Wider rows: the same, with the row read again for its norm and for its codes.
template <typename T, bool BYTES>
__global__ void quantized_norm_kernel(const QnArgs a) {
  pdl_trigger();      // (see microscaled_rows_kernel)
  pdl_wait();
  __shared__ float scratch[32];
  __shared__ uint32_t scratch_max[32];
  const int orow = blockIdx.x, srow = qn_row(a, orow);
  const float* res = a.residual + (size_t)srow * a.hidden;
  const T* delta = a.delta ? static_cast<const T*>(a.delta) + (size_t)srow * a.hidden : nullptr;
  // (h is added up anew where it is needed: residual and sum may be the same memory, where each thread reads and writes the columns of its own)
  float* sum = a.sum ? a.sum + (size_t)srow * a.hidden : nullptr;
  const bool kept = sum != nullptr;
  float ss = 0.f;
  for (int c = threadIdx.x; c < a.hidden; c += blockDim.x) {
    float h = res[c];
    if (delta) h += to_f32(delta[c]);
    if (kept) sum[c] = h;
    ss += h * h;
  }
  const float total = qn_block_sum(ss, scratch);      // (its barrier makes the block's sums readable to all of it)
  const float inv = rsqrtf(total / (float)a.hidden + a.eps);
  auto normed = [&](int c) {
    if (c >= a.hidden) return 0.f;
    float h = kept ? sum[c] : res[c];
    if (!kept && delta) h += to_f32(delta[c]);
    return to_f32(from_f32<T>(h * inv * a.weight[c]));
  };
  uint32_t largest = 0;
  T* out = a.out ? static_cast<T*>(a.out) + (size_t)orow * a.hidden : nullptr;
  if (!BYTES || out)
    for (int c = threadIdx.x; c < a.hidden; c += blockDim.x) {
      const float v = normed(c);
      largest = max(largest, __float_as_uint(v) & 0x7fffffffu);
      if (out) out[c] = from_f32<T>(v);
    }
  float r = 1.f, inverse = 1.f;
  if constexpr (!BYTES) ms_row_scale(qn_block_max(largest, scratch_max), r, inverse);
  const int steps = (a.hidden + kMsStep - 1) / kMsStep, eights = steps * (kMsStep / 8);
  for (int g = threadIdx.x; g < eights; g += blockDim.x) {      // (whole warps: both are multiples of 32)
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = normed(g * 8 + i);
    qn_codes8<T, BYTES>(a, orow, g, v, r, inverse, steps);
  }
}

// Rows of more than 8,192 columns take 33 to 64 KB, and the kernel's own arrays beside them: above the 48 KB that it has without asking from 12,036 columns on.  It asks once a
// device (the attribute belongs to its context), whatever the row's width.
template <typename T, bool BYTES>
static int qn_allow_smem(void (*kern)(const QnArgs, int)) {
  static bool allowed[64];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && !(device < 64 && allowed[device])) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kQnFoursWidth * (int)sizeof(float));
  if (e != cudaSuccess) return (int)e;
  if (device < 64) allowed[device] = true;
  return TIB_OK;
}

}  // namespace tib

using namespace tib;

// residual [n_rows, hidden] fp32, delta [n_rows, hidden] in dtype or null; sum [n_rows, hidden] fp32 takes residual + delta (it may be residual itself, or an fp32 delta; null: it is not kept, and
// with `rows`, indices of the n_out rows to norm, it has to be null).  bytes 0: codes, scales, factors as tib_microscaled_rows leaves them, 1: codes
// [n_out, runs * 128] and factors = scales [runs, lds] as tib_quantize_rows does.  out: the normed rows in dtype, or null, memory of its own.
TIB_API int tib_quantized_norm(const void* delta, const float* residual, float* sum, const int* rows, const float* weight, void* out, int bytes, void* codes,
                               void* scales, float* factors, int64_t lds, int n_out, int n_rows, int hidden, float eps, int dtype, cudaStream_t stream) {
  if (n_out == 0) return TIB_OK;
  if (!residual || !weight || !codes || !factors || (!bytes && !scales) || n_out < 0 || n_rows < 1 || (!rows && n_out > n_rows) || hidden < 1 || (rows && sum)) return TIB_E_ARG;
  if (dtype != TIB_BF16 && dtype != TIB_F32) return TIB_E_DTYPE;
  if (bytes && lds < n_out) return TIB_E_SIZE;
  if (((uintptr_t)codes | (uintptr_t)scales) & 15) return TIB_E_ALIGN;
  // (a block writes its row's sum and normed form while others read theirs)
  const int64_t size = dtype == TIB_BF16 ? 2 : 4, numbers = (int64_t)n_rows * hidden, normed = (int64_t)n_out * hidden;
  auto share = [](const void* p, int64_t p_bytes, const void* q, int64_t q_bytes) { return p && q && (const char*)p < (const char*)q + q_bytes && (const char*)q < (const char*)p + p_bytes; };
  if ((sum != residual && share(sum, 4 * numbers, residual, 4 * numbers)) || (!(sum == delta && size == 4) && share(sum, 4 * numbers, delta, size * numbers)) ||
      share(sum, 4 * numbers, weight, (int64_t)4 * hidden) || share(out, size * normed, residual, 4 * numbers) || share(out, size * normed, delta, size * numbers) ||
      share(out, size * normed, sum, 4 * numbers) || share(out, size * normed, weight, (int64_t)4 * hidden))
    return TIB_E_OVERLAP;
  const QnArgs a{delta, residual, sum, rows, weight, out, (unsigned char*)codes, (unsigned char*)scales, factors, lds, hidden, eps, ms_groups(n_out, 0), n_rows};
  if (dtype == TIB_BF16 && hidden % 8 == 0 && hidden <= 8192 &&
      (((uintptr_t)residual | (uintptr_t)sum | (uintptr_t)weight | (uintptr_t)out | (uintptr_t)delta) & 15) == 0) {
    const int threads = (hidden / 8 + 31) / 32 * 32;
    if (bytes) TIB_LAUNCH_DEPENDENT(quantized_norm_bf16x8_kernel<true>, n_out, threads, 0, stream, a);
    else TIB_LAUNCH_DEPENDENT(quantized_norm_bf16x8_kernel<false>, n_out, threads, 0, stream, a);
    return TIB_OK;
  }
  const int threads = norm_threads(hidden);
  const size_t smem = (size_t)ceil_div(hidden, kMsStep) * kMsStep * sizeof(float);
  if (hidden % 4 == 0 && hidden <= kQnFoursWidth && (((uintptr_t)residual | (uintptr_t)sum | (uintptr_t)weight | (uintptr_t)out | (uintptr_t)delta) & 15) == 0) {
    const int quarter = (threads / 4 + 31) / 32 * 32, held = ceil_div(hidden, threads);      // (at most 16: threads is hidden / 4 or 1,024)
#define TIB_QN_X4(T, BYTES, HELD)                                                                                                          \
  do {                                                                                                                                     \
    auto kern = quantized_norm_x4_kernel<T, BYTES, HELD>;                                                                                  \
    if (HELD == 16) {                                                                                                                      \
      const int rc = qn_allow_smem<T, BYTES>(kern);                                                                                        \
      if (rc != TIB_OK) return rc;                                                                                                         \
    }                                                                                                                                      \
    TIB_LAUNCH_DEPENDENT(kern, n_out, quarter, smem, stream, a, threads);                                                                  \
  } while (0)
#define TIB_QN_X4_HELD(T, BYTES)                 \
  do {                                           \
    if (held <= 4) TIB_QN_X4(T, BYTES, 4);       \
    else if (held <= 8) TIB_QN_X4(T, BYTES, 8);  \
    else TIB_QN_X4(T, BYTES, 16);                \
  } while (0)
    if (dtype == TIB_BF16) {
      if (bytes) TIB_QN_X4_HELD(__nv_bfloat16, true);
      else TIB_QN_X4_HELD(__nv_bfloat16, false);
    } else {
      if (bytes) TIB_QN_X4_HELD(float, true);
      else TIB_QN_X4_HELD(float, false);
    }
#undef TIB_QN_X4_HELD
#undef TIB_QN_X4
    return TIB_OK;
  }
#define TIB_QN_GO(T, BYTES)                                                                                                  \
  do {                                                                                                                       \
    if (hidden <= kQnWidth) TIB_LAUNCH_DEPENDENT((quantized_norm_held_kernel<T, BYTES>), n_out, threads, smem, stream, a);   \
    else TIB_LAUNCH_DEPENDENT((quantized_norm_kernel<T, BYTES>), n_out, threads, 0, stream, a);                              \
  } while (0)
  if (dtype == TIB_BF16) {
    if (bytes) TIB_QN_GO(__nv_bfloat16, true);
    else TIB_QN_GO(__nv_bfloat16, false);
  } else {
    if (bytes) TIB_QN_GO(float, true);
    else TIB_QN_GO(float, false);
  }
#undef TIB_QN_GO
  return TIB_OK;
}

TIB_PACKED(tib_quantized_norm)
