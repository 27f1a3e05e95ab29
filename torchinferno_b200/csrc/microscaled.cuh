// What the kernels of 4-bit microscaled operands share.
//
// A code is an e2m1 number (a sign, two bits of exponent, one of mantissa: 0, 1/2, 1, 3/2, 2, 3, 4, 6), two in a byte, the even column in the lower half.
// Sixteen columns have one e4m3 scale (never negative).  A matrix [N, K] has one fp32 factor, held for each of its rows; rows x [M, K] have a power
// of two each.  Columns are padded with zeros to whole steps of 256 (128 bytes of codes, the row of the 128-byte swizzle; four MMAs of 64 columns).
// Codes lie as the MMA reads them from shared memory, eight rows' 128 bytes of a step side by side, the 16-byte piece p of row i at p ^ (i % 8) (the 128-byte
// swizzle), so that plain copies bring them.
//   codes of a matrix   [tiles of 128 rows][steps][16 groups of 8 rows][1024 bytes]: a step's 16 KB of a tile are one copy
//   codes of rows       [steps][groups of 8 rows][1024 bytes]: a step of neighbouring rows is one copy
//   scales of both      [tiles of 128 rows][steps][4 chunks of 64 columns][512 bytes], row i of a tile at (i % 32) * 16 + (i / 32) * 4, a byte for each run of
//                       16 columns: a chunk is what one tcgen05.cp of 32 x 128 bits brings to tensor memory, where lane i % 32 of column i / 32 then
//                       holds the four scales of row i
// The groups (and the scales' tiles) of rows sorted by expert begin with the experts' first rows: expert e, whose rows begin at o_e, has those from
// ceil(o_e / 8) + e (ceil(o_e / 128) + e) on.  (o_e + n_e = o_(e + 1), so these end before the next expert's begin; all are fewer than ceil(M / 8) +
// experts.)
#pragma once

#include "block_scaled.cuh"
#include "cluster.cuh"

namespace tib {

constexpr int kMsRun = 16, kMsStep = 256, kMsStepBytes = 128, kMsChunkBytes = 512, kMsStepScales = 4 * kMsChunkBytes, kMsTileRows = 128;
constexpr int kMsGroup = 8, kMsGroupBytes = kMsGroup * kMsStepBytes;

static inline int ms_steps(int K) { return ceil_div(K, kMsStep); }
__host__ __device__ __forceinline__ int ms_first_tile(int first_row, int expert) { return ((first_row + kMsTileRows - 1) >> 7) + expert; }
__host__ __device__ __forceinline__ int ms_first_group(int first_row, int expert) { return ((first_row + kMsGroup - 1) >> 3) + expert; }
static inline int ms_groups(int M, int experts) { return ceil_div(M, kMsGroup) + experts; }      // (experts: 0 for rows that are not sorted)
// the place of byte b (0 .. 127) of a step of row i of a group, in the group
__host__ __device__ __forceinline__ int ms_code_at(int i, int b) { return (i << 7) + ((((b >> 4) ^ i) << 4) | (b & 15)); }
// the place of row i of a tile's four scales of a chunk
__host__ __device__ __forceinline__ int ms_scale_at(int i) { return ((i & 31) << 4) + ((i >> 5) << 2); }

// A row whose largest absolute value has these bits: 2^p and 2^-p, p the smallest integer, at least -126, for which the largest is at most 2688 * 2^p (2688 =
// 6 * 448 = 1.3125 * 2^11: the largest code times the largest scale); 1 for a row of zeros.  A power of two divides without rounding and leaves
// the scales their three bits of mantissa over the 17 binades of e4m3.  A row that holds an infinity or a NaN gets a NaN, which shows in every output, and codes of 0.
__device__ __forceinline__ void ms_row_scale(uint32_t largest, float& r, float& inverse) {
  int p = (int)(largest >> 23) - 127 - 11 + ((largest & 0x7fffffu) > 0x280000u);
  p = p < -126 ? -126 : p;
  if (largest == 0) p = 0;
  r = __uint_as_float((uint32_t)(p + 127) << 23);
  inverse = __uint_as_float((uint32_t)(127 - p) << 23);
  if (largest >= 0x7f800000u) { r = __uint_as_float(0x7fc00000u); inverse = 0.f; }
}

// Quotients are made with an approximate reciprocal and still rounded as the exact quotient is.  A border between two codes (or two scales) times the divisor has at
// most seven significant bits, so a number of up to twelve is either on the border or off by 2^-12 of it, far more than the 2^-22 that the
// product with the reciprocal is off by: rounded to 16 bits, or to multiples of 2^-16 (a border of codes is 1/4 or more), it is on the border if and only if the exact
// quotient is.  A bf16 has eight bits; a 32-bit number is first cut to twelve, the last of them set where any that was cut off is (which leaves it on the same side of
// every number of fewer bits).  That holds for normal numbers: a subnormal one that may be near a border is multiplied by 2^32 before it is cut (ms_codes8).
template <typename T> __device__ __forceinline__ float ms_odd12(float v) {
  if constexpr (sizeof(T) == 2) return v;
  const uint32_t b = __float_as_uint(v);
  return __uint_as_float((b & 0xfffff000u) | (((b & 0xfffu) + 0xfffu) & 0x1000u));
}
__device__ __forceinline__ float ms_round16(float v) { return __uint_as_float((__float_as_uint(v) + 0x80u) & 0xffffff00u); }

// The scale of a run whose largest number, times the row's inverse, is t: its e4m3 code; and what it stands for.
template <typename T> __device__ __forceinline__ uint32_t ms_run_scale(float t) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(ms_round16(ms_odd12<T>(t) * (1.f / 6.f))));
  return r & 0xffu;
}
__device__ __forceinline__ float ms_scale_value(uint32_t code) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}
__device__ __forceinline__ float ms_reciprocal(float s) {      // 0 for 0
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return s == 0.f ? 0.f : r;
}
// Eight numbers times `inverse` (a power of two) and `reciprocal` to eight codes, the first in the lowest four bits.  (The two factors are one where their product
// is a normal number: but for rows whose largest number is under 2^-97, of which the numbers are multiplied by 2^32 first, so that none near a border is
// subnormal.  In other rows r is 2^-108 or more and the least scale 2^-9: a subnormal number is less than 2^-9 of that, and its code 0, cut or not.)
template <typename T> __device__ __forceinline__ uint32_t ms_codes8(const float (&numbers)[8], float inverse, float reciprocal) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = numbers[j];
  if (inverse > 0x1p108f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= 0x1p32f;
    inverse *= 0x1p-32f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = ms_odd12<T>(v[j]);
  // (192 + q is a multiple of 2^-16; a quotient is at most 9, where a scale of 1.5 * 2^-9 was rounded to 2^-9)
  const f32x2 factor = f2_pack(inverse * reciprocal, inverse * reciprocal), up = f2_pack(192.f, 192.f), down = f2_pack(-192.f, -192.f), one = f2_pack(1.f, 1.f);
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) f2_unpack(f2_fma(f2_fma(f2_pack(v[j], v[j + 1]), factor, up), one, down), q[j], q[j + 1]);
  uint32_t codes;
  asm("{\n.reg .b8 a, b, c, d;\ncvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\ncvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\nmov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(codes) : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return codes;
}
// A run's codes and (into `scale`) its scale.  inverse: of the row's factor, 0 where the row holds no finite sum.
template <typename T> __device__ __forceinline__ uint2 ms_run_codes(const uint4 (&raw)[sizeof(T)], uint32_t run_largest, float inverse, uint32_t& scale) {
  const float t = __uint_as_float(run_largest) * inverse;
  scale = inverse == 0.f ? 0u : ms_run_scale<T>(t);
  const float reciprocal = ms_reciprocal(ms_scale_value(scale));
  float v[16], lo[8], hi[8];
  bs_floats16<T>(raw, v);
#pragma unroll
  for (int j = 0; j < 8; ++j) lo[j] = v[j], hi[j] = v[8 + j];
  return scale == 0 ? make_uint2(0, 0) : make_uint2(ms_codes8<T>(lo, inverse, reciprocal), ms_codes8<T>(hi, inverse, reciprocal));
}
// two codes (a byte) to two floats
__device__ __forceinline__ float2 ms_numbers2(uint32_t byte) {
  uint32_t h;
  asm("{\n.reg .b8 b;\ncvt.u8.u32 b, %1;\ncvt.rn.f16x2.e2m1x2 %0, b;\n}\n" : "=r"(h) : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// D fp32 in tensor memory (+)= the product of a chunk's 64 columns: A and B e2m1 in shared memory, K-major (descriptors by their lower halves), each
// row's four e4m3 scales in tensor memory.  The instruction descriptor but for N and M: both types e2m1, unsigned e4m3 scales.
constexpr uint32_t kMsIdesc = (1u << 7) | (1u << 10);
// By one elected thread, in a branch of its own: predicated by lane, as the products of other kernels are, a copy took 45 cycles of the warp that issues it and an
// MMA 64, and sixteen of them a step were what bound it (8,192 rows 8,192 -> 28,672: 1,118 us, in a branch 674).
template <int CTAS>
__device__ __forceinline__ void ms_umma(uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, uint32_t accumulate) {
  static_assert(CTAS == 1 || CTAS == 2, "blocks of a tile");
  if constexpr (CTAS == 1)
    asm volatile("{\n.reg .pred p;\n.reg .b64 a, b;\nmov.b64 a, {%1, %7};\nmov.b64 b, {%2, %7};\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], a, b, %3, [%4], [%5], p;\n}\n"
                 ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate), "r"(kUmmaDescHigh) : "memory");
  else
    asm volatile("{\n.reg .pred p;\n.reg .b64 a, b;\nmov.b64 a, {%1, %7};\nmov.b64 b, {%2, %7};\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], a, b, %3, [%4], [%5], p;\n}\n"
                 ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate), "r"(kUmmaDescHigh) : "memory");
}
// A chunk's scales (512 bytes of shared memory: 32 rows of 16) to four columns of tensor memory, once for each of its four groups of lanes.  The descriptor: no
// swizzle, groups of eight rows 128 bytes apart.
template <int CTAS> __device__ __forceinline__ void ms_copy_scales(uint32_t tmem, uint32_t smem) {
  const uint32_t low = (smem & 0x3FFFF) >> 4, high = (128u >> 4) | (1u << 14);
  if constexpr (CTAS == 1)
    asm volatile("{\n.reg .b64 s;\nmov.b64 s, {%1, %2};\ntcgen05.cp.cta_group::1.32x128b.warpx4 [%0], s;\n}\n" ::"r"(tmem), "r"(low), "r"(high) : "memory");
  else
    asm volatile("{\n.reg .b64 s;\nmov.b64 s, {%1, %2};\ntcgen05.cp.cta_group::2.32x128b.warpx4 [%0], s;\n}\n" ::"r"(tmem), "r"(low), "r"(high) : "memory");
}
// Bytes side by side in memory to shared memory (both 16-byte aligned, a multiple of 16), counted on a barrier.
__device__ __forceinline__ void ms_bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// The rows of a product: x as codes.
struct MsRows {
  const unsigned char* codes;      // [steps, groups, 1024]
  const unsigned char* scales;     // [tiles, steps, 2048]
  const float* factors;            // [M]
  int groups;
};

// A product's arguments.
struct MsArgs {
  MsRows x;
  const unsigned char* w;          // codes of the matrices
  const unsigned char* w_scales;
  const float* w_factors;          // [experts, N]
  int M, N, steps, stages, tmem_cols;
  const int* offsets;              // [experts + 1] of rows sorted by expert, or null: one matrix
  const int* order;
  int experts;
  float limit, alpha;              // of the clamped gated unit
  const float* row_scale;          // [M] by pair, or null
  int* error_word;
  const __nv_bfloat16* made;       // the rows themselves where the product's kernel makes their codes (then `x` is empty), or null
  int64_t ld_made;
  int K;
};

// An output is sum * f * r * q: the matrix's factor f, the row's power of two r (or NaN) and its pair's factor q (1 where it has none).  A sum is 0 or from 2^-20 (two codes
// of 1/2, two scales of 2^-9) to under 2^56 in size.  The kernels take the products in an order in which nothing leaves the range of 32 bits but what the output itself does,
// for q from 2^-50 to 2^50 in size or 0 and
//   f from 2^-100 to 2^70 (or 0), which leaves every sum a normal number: f first, then what ms_row_scales gives.  (In the fewest steps: microscaled_tcgen05.cu.  With what
//   follows in their place 8 rows 1,024 -> 1,024 took 4.2 us for 3.95, with a branch for other factors as much.)
//   any f: what ms_row_factors gives, ahead of f and behind it (microscaled_2cta.cu, where it costs nothing; matrices with other factors run there whatever their rows are).
// Behind an ordinary f: r q, exact where it is a normal number.  Where it is too small for one, q is less than 1 (r is 2^-126 or more), and where it is too large, more
// (r is 2^117 or less): then r comes first, and what leaves the range with it does so with both.
__device__ __forceinline__ float2 ms_row_scales(float r, float q) {
  const float both = r * q;
  return (fabsf(both) >= 0x1p-126f && fabsf(both) < INFINITY) || q == 0.f ? make_float2(both, 1.f) : make_float2(r, q);
}
// With q = m 2^e, 1 <= m < 2, what comes ahead of f is the power of two 2^e r, kept within 2^-106 .. 2^70, where it leaves every sum a normal number, and exact; what it was kept
// from comes behind f, with m.  So if the product with f is too large, so is the output (what is left is at least 1), and if that is too small to be a normal number, the
// output is, too (what is left is less than 2).
__device__ __forceinline__ float2 ms_row_factors(float r) {      // (q = 1; a NaN is behind)
  const float first = fminf(fmaxf(r, 0x1p-106f), 0x1p70f);
  return make_float2(first, first == r ? 1.f : r * (r > 1.f ? 0x1p-70f : 0x1p106f));
}
__device__ __forceinline__ float2 ms_row_factors(float r, float q) {
  if (!(r < INFINITY && fabsf(q) < INFINITY) || q == 0.f) return make_float2(q == 0.f ? 0.f : 1.f, r * q);
  int e = (int)(__float_as_uint(r) >> 23) - 2 * 127;
  if (fabsf(q) < 0x1p-126f) q *= 0x1p24f, e -= 24;
  const uint32_t bits = __float_as_uint(q);
  e += (int)((bits >> 23) & 0xffu);
  const int first = min(max(e, -106), 70), last = min(max(e - first, -126), 127);
  return make_float2(__uint_as_float((uint32_t)(first + 127) << 23), __uint_as_float((bits & 0x807fffffu) | 0x3f800000u) * __uint_as_float((uint32_t)(last + 127) << 23));
}

// Products of rows that are there as codes (microscaled_tcgen05.cu, microscaled_2cta.cu), with arguments that tib_microscaled_product has checked.
bool ms_on_pairs_of_sms(int M, int N, int steps, int experts);
int ms_product_2cta(const MsArgs& a, int act, void* y, int y_dtype, int64_t ldy, cudaStream_t stream);
// How a product runs there: {rows of a tile at most, blocks that share a tile, steps of a block at most, stages of its ring}.
int ms_plan_2cta(int M, int N, int steps, int experts, int* plan);
int ms_plan_tcgen05(int M, int N, int steps, int experts, int* plan);
// What a block of it takes: {columns of tensor memory, bytes of shared memory}.
int ms_room_2cta(int experts, int* room);
int ms_room_tcgen05(int M, int N, int steps, int experts, int* room);
// Whether the kernel of a product with one matrix may make the codes of its rows itself.
bool ms_makes_rows(int M, int N, int K);
int ms_product_tcgen05(MsArgs& a, int act, void* y, int y_dtype, int64_t ldy, cudaStream_t stream);

}  // namespace tib
