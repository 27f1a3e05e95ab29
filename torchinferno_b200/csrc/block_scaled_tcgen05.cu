// Products of 8-bit block-scaled operands on the 5th-generation tensor cores, for few rows and for rows sorted by expert:
//     y[m, n] = act(sum over runs b of s[m, b] S[n's block, b] (sum over the 128 columns of run b of x[m, k] w[n, k]))
//
// The weights are the 128-row operand of the MMA and the rows its N dimension: a tile is 128 features x up to NT rows, the rows rounded up to 16
// only, and the accumulator is the transposed output (TMEM lane = feature, column = row).  A step of the loop is one run: 128 columns, the 128-byte
// row of the swizzle, four MMAs into an accumulator of its own in tensor memory, which the summing warps take out and add to 32-bit sums in
// registers, times the scale of (row, run) and (block of features, run), whose product is made once a row and step (packed fp32, one multiply-add for
// two sums).  kBufs accumulators rotate, so the tensor cores run ahead of the sums.
//   warp 0             TMA producer: 16 KB of codes of w a step, one block of the matrix, and the rows' codes where they exist, in boxes of 32 rows
//   warp 1             issues tcgen05.mma; owns the TMEM allocation
//   the next 4 or 8    sums and epilogue (eight for 128 rows: four for each half of the columns)
//   the last 2 or 4    helpers, taking turns: the products of scales into a ring of their own; from rows that are no codes yet they (then four) make
//                      these, straight into the swizzled stage (a step of few rows then has no kernel ahead of its products)
// A summing thread takes two columns in eight of four features (tcgen05.ld 16x256b), and so reads a quarter of a step's scales: shared memory is what
// the MMAs of 128 x 128 x 128 wait for (their operands and the copies that bring them take it for 512 of a step's cycles, the tensor cores 256).
// A matrix of few tiles is split by runs over a cluster of up to eight blocks, whose sums meet in distributed shared memory, added in the
// blocks' order.  Weights do not depend on the kernel before: a first ring of them is requested before griddepcontrol.wait (not for sorted rows, whose
// tiles that kernel's counts decide).
//
// What bounds it, at few rows: memory.  8 rows 4,096 -> 2 x 14,336: 21.2 us for 117 MB (5.5 TB/s, 84 % of the measured copy bandwidth; two blocks an SM: with one,
// whose second round of tiles is half empty, 31); 14,336 -> 4,096 13.7 to 14.1 us for 59 MB; 21 of 32 experts' 88 MB 14.3 us.  One row 4,096 -> 4,096 takes 7.6 us for
// the 2.6 of its stream: about 3,000 cycles pass between the kernel before's end and the first sums, 1,400 in the exchange, 1,100 at the end, and one SM's share of the
// launch is 1.4 us.  In tiles of 128 rows shared memory, in smaller ones the summing warps' loop (300 to 400 cycles a step).  Every wait is bounded and reports in
// error_word; a warp that gave up goes through the motions to the end, so that nobody waits for it.
#include "block_scaled.cuh"
#include "mma.cuh"
#include "cluster.cuh"

namespace tib {

constexpr int kBsMaxExperts = 1024, kBsMaxStages = 16, kBsSlots = 16;      // (slots: of the ring of scales)
constexpr uint32_t kBsBarBytes = 640;
constexpr uint32_t kBsWBytes = 128 * kBlk;

template <int NT, bool CODES> struct BsShape {
  static constexpr int kStorers = NT >= 128 ? 8 : 4, kHelpers = CODES ? 2 : 4, kThreads = 64 + 32 * (kStorers + kHelpers);
  static constexpr int kPerSm = NT <= 32 ? 2 : 1;                   // blocks of an SM
  static constexpr int kBufs = 4, kCols = NT / (kStorers / 4);      // accumulators; columns of a summing thread
  static constexpr uint32_t kTmemCols = kBufs * NT < 32 ? 32 : kBufs * NT;
  static constexpr uint32_t kStage = kBsWBytes + NT * kBlk;
  static constexpr int kScales = 2 * NT + 8;                        // of a step: for even features, behind them for odd ones (on other banks)
};

// (a column's 128 / splits sums and four more: the eight features and four columns that a warp writes at a time then fall on all banks)
template <int NT> __host__ __device__ constexpr int bs_red_floats(int splits) { return NT * (128 + 4 * splits); }

struct BsTile { int expert, first, rows, feature; };

struct BsArgs {
  const void* x;               // codes [rows, runs * 128], or rows of the activations' type
  int64_t ldx;                 // (of the latter)
  const float* x_scales;       // [runs, lds] beside codes
  const unsigned char* w;      // codes in blocks
  const float* w_scales;       // [experts, scale_rows, runs]
  int scale_rows, pairs, vec, lds;       // vec: rows of x are 16-byte aligned
  int M, N, K, runs, x_rows, stages;
  const int* offsets;          // null: one matrix
  const int* order;
  int experts, top, modes;     // modes: kBsByPair, kBsWide
  float far_low;               // (BsFar)
  int act;
  float limit, alpha, far_high;
  const float* row_scale;
  int* error_word;

  __device__ __forceinline__ bool outside(float s) const { return BsFar{far_low, far_high}.outside(s); }
};
constexpr int kBsByPair = 1, kBsWide = 2;      // a row of x is a token's, not a pair's; rows of y are 16-byte aligned
// (Two tensor maps, these, y and its stride.  On the host a launch with more than 416 bytes takes 0.3 us of 2.8 more; on the device flags packed into bits of one word
// cost 0.1 us of 5 to 14 at few rows.)
static_assert(2 * sizeof(CUtensorMap) + sizeof(BsArgs) + 16 <= 416, "the kernel's parameters");

__device__ __forceinline__ int bs_source(const BsArgs& a, const BsTile& m, int r) {      // the row of x that the tile's row r is
  const int at = m.first + min(r, m.rows - 1);
  return a.offsets && (a.modes & kBsByPair) ? min(bs_pair(a.order, at, a.M) / a.top, a.x_rows - 1) : at;
}

__device__ __forceinline__ void umma_f8_warp(uint32_t leader, uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p, q;\n.reg .b64 a, b;\nmov.b64 a, {%1, %6};\nmov.b64 b, {%2, %6};\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
               "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n}\n"
               ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(leader), "r"(kUmmaDescHigh) : "memory");
}
// 16 lanes of tensor memory, COLS columns of them: register 4 j + 2 h + i is lane (thread / 4) + 8 h, column 8 j + 2 (thread % 4) + i
template <int COLS> __device__ __forceinline__ void tmem_ld_16x256b(uint32_t taddr, uint32_t (&r)[COLS / 2]) {
  static_assert(COLS == 16 || COLS == 32 || COLS == 64, "columns");
  if constexpr (COLS == 16)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
  else if constexpr (COLS == 32)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr));
  else
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(taddr));
}
__device__ __forceinline__ void bs_fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// A block's share of a tile from its sums in shared memory (and the other blocks' beside them) through the activation to y: eight outputs of a
// column a thread and turn.  A function for each activation: with the choice inside the loop a turn took 1,250 cycles, most of them fetching code.
template <int ACT, int NT, typename TO>
__device__ __forceinline__ void bs_finish(const float* red, int log_splits, int rank, const BsTile& m, const BsArgs& a, TO* __restrict__ y, int64_t ldy,
                                          int thread, int threads) {
  constexpr int kGated = moe_act_gated(ACT);
  const int per = 128 >> log_splits, stride = per + 4, splits = 1 << log_splits;
  const int log_wide = 4 - log_splits - kGated;           // eights of outputs in a column
  const int first_out = (m.feature + rank * per) >> kGated, n_out = a.N >> kGated;
  if (!(a.modes & kBsWide)) {
    // Rows of y that are not 16-byte aligned: a warp takes a row, its lanes consecutive outputs.
    const int lane = thread & 31, outs = per >> kGated;
#pragma unroll 1
    for (int c = thread >> 5; c < m.rows; c += threads >> 5) {
      const float scale = a.row_scale ? a.row_scale[bs_pair(a.order, m.first + c, a.M)] : 1.f;
      TO* dst = y + (size_t)(m.first + c) * ldy + first_out;
#pragma unroll
      for (int j = 0; j < 4 >> kGated; ++j) {
        const int o = 32 * j + lane;
        if (o >= outs) break;
        const float* from = red + c * stride + (o << kGated);
        float g = from[0], u = from[kGated];
        for (int r = 1; r < splits; ++r) {
          from += NT * stride;
          g += from[0];
          u += from[kGated];
        }
        g *= scale;
        if (first_out + o < n_out) dst[o] = from_f32<TO>(kGated ? bs_gated<ACT>(g, u * scale, a.limit, a.alpha) : bs_act<ACT>(g));
      }
    }
    return;
  }
#pragma unroll 1
  for (int i = thread; i < m.rows << log_wide; i += threads) {
    const int c = i >> log_wide, f = (i - (c << log_wide)) * 8;
    if (first_out + f >= n_out) continue;
    float v[8 << kGated];
    const float* from = red + c * stride + (f << kGated);
#pragma unroll
    for (int j = 0; j < 8 << kGated; j += 4) {
      const float4 p = *reinterpret_cast<const float4*>(from + j);
      v[j] = p.x; v[j + 1] = p.y; v[j + 2] = p.z; v[j + 3] = p.w;
    }
    for (int r = 1; r < splits; ++r) {
      from += NT * stride;
#pragma unroll
      for (int j = 0; j < 8 << kGated; j += 4) {
        const float4 p = *reinterpret_cast<const float4*>(from + j);
        v[j] += p.x; v[j + 1] += p.y; v[j + 2] += p.z; v[j + 3] += p.w;
      }
    }
    if (a.row_scale) {
      const float scale = a.row_scale[bs_pair(a.order, m.first + c, a.M)];
#pragma unroll
      for (int j = 0; j < 8 << kGated; ++j) v[j] *= scale;
    }
    float out[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (kGated) out[j] = bs_gated<ACT>(v[2 * j], v[2 * j + 1], a.limit, a.alpha);
      else out[j] = bs_act<ACT>(v[j]);
    }
    TO* dst = y + (size_t)(m.first + c) * ldy + first_out + f;
    if (first_out + f + 8 <= n_out) {
      if constexpr (sizeof(TO) == 2) {
        __nv_bfloat162 p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(out[2 * j], out[2 * j + 1]);
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(p);
      } else {
        reinterpret_cast<float4*>(dst)[0] = make_float4(out[0], out[1], out[2], out[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(out[4], out[5], out[6], out[7]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (first_out + f + j < n_out) dst[j] = from_f32<TO>(out[j]);
    }
  }
}

// The outputs of a block's share of a tile that have a far scale, made again by a warp.
template <typename TX, typename TO>
__device__ __forceinline__ void bs_tile_apart(const BsArgs& a, const BsTile& m, int rank, int splits, int lane, TO* __restrict__ y, int64_t ldy) {
  constexpr bool kCodes = std::is_same_v<TX, uint8_t>;
  const int gated = moe_act_gated(a.act) ? 1 : 0, outs = 128 / splits >> gated, first = (m.feature >> gated) + rank * outs, n_out = a.N >> gated;
#pragma unroll 1
  for (int c = 0; c < m.rows; ++c) {
    BsApart<TX> apart;
    apart.x = static_cast<const TX*>(a.x) + (kCodes ? (size_t)(m.first + c) * a.runs * kBlk : (size_t)bs_source(a, m, c) * a.ldx);
    apart.x_scales = a.x_scales + (kCodes ? m.first + c : 0);
    apart.lds = a.lds; apart.pairs = a.pairs; apart.runs = a.runs; apart.K = a.K; apart.act = a.act;
    apart.limit = a.limit; apart.alpha = a.alpha;
    bool outside = false;
    for (int kb = lane; kb < a.runs; kb += 32) {
      float inverse;
      outside |= a.outside(apart.run_scale(kb, inverse));
    }
    if (!__any_sync(0xffffffffu, outside)) continue;
    apart.row_scale = a.row_scale ? a.row_scale[bs_pair(a.order, m.first + c, a.M)] : 1.f;
    apart.w = a.w + ((size_t)m.expert * ((a.N + 127) >> 7) * a.runs << 14);
    apart.w_scales = a.w_scales + (size_t)m.expert * a.scale_rows * a.runs;
    for (int o = first + lane; o < min(first + outs, n_out); o += 32) bs_output_apart<TX, TO>(apart, o, y + (size_t)(m.first + c) * ldy);
  }
}

template <int NT, typename TX, typename TO>
__global__ void __launch_bounds__(BsShape<NT, std::is_same_v<TX, uint8_t>>::kThreads, BsShape<NT, std::is_same_v<TX, uint8_t>>::kPerSm)
block_scaled_tcgen05_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const BsArgs a,
                            TO* __restrict__ y, int64_t ldy) {
  constexpr bool kCodes = std::is_same_v<TX, uint8_t>;
  using S = BsShape<NT, kCodes>;
  const int splits = NT >= 128 ? 1 : (int)cluster_size(), rank = NT >= 128 ? 0 : (int)cluster_rank();
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem_gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + a.stages * S::kStage;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kBsMaxStages + s); };
  auto acc_full_bar = [&](int b) { return bars + 8u * (2 * kBsMaxStages + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * kBsMaxStages + S::kBufs + b); };
  auto scale_full_bar = [&](int i) { return bars + 8u * (2 * kBsMaxStages + 2 * S::kBufs + i); };
  auto scale_empty_bar = [&](int slot) { return bars + 8u * (2 * kBsMaxStages + 2 * S::kBufs + kBsSlots + slot / 4); };      // (four slots are freed together)
  const uint32_t red_bar = bars + 8u * (2 * kBsMaxStages + 2 * S::kBufs + kBsSlots + kBsSlots / 4), tmem_slot = red_bar + 8, far_seen = red_bar + 12;      // (not 0: some row's scale is outside, BsFar)
  static_assert(8 * (2 * kBsMaxStages + 2 * S::kBufs + kBsSlots + kBsSlots / 4) + 16 <= kBsBarBytes, "the barriers' share of shared memory");
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_gen + (tmem_slot - base));
  float* step_scales = reinterpret_cast<float*>(smem_gen + (bars - base) + kBsBarBytes);  // [kBsSlots][kScales]
  float* red = step_scales + kBsSlots * S::kScales;                                       // [splits][NT][128 / splits + 4] sums
  int* tiles_before = reinterpret_cast<int*>(red + bs_red_floats<NT>(splits));            // [experts + 1] where rows are sorted, and
  int* first_row = tiles_before + a.experts + 1;                                          // [experts + 1] their offsets

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int cluster_id = blockIdx.x / splits, clusters = gridDim.x / splits;
  const int kb0 = (int)((int64_t)a.runs * rank / splits), kb1 = (int)((int64_t)a.runs * (rank + 1) / splits);
  if (warp == 0) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map_w) : "memory");
      if constexpr (kCodes) asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map_x) : "memory");
    }
    if (lane < a.stages) {
      mbar_init(full_bar(lane), kCodes ? 1 : 2);  // the producer, and the helper that makes codes
      mbar_init(empty_bar(lane), 1);
    }
    if (lane < kBsSlots) mbar_init(scale_full_bar(lane), 1);
    if (lane < kBsSlots / 4) mbar_init(scale_empty_bar(4 * lane), S::kStorers);
    if (lane < S::kBufs) {
      mbar_init(acc_full_bar(lane), 1);
      mbar_init(acc_empty_bar(lane), S::kStorers);
    }
    if (lane == 0) {
      mbar_init(red_bar, 1);
      *reinterpret_cast<uint32_t*>(smem_gen + (far_seen - base)) = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tmem_slot), "r"(S::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (a.offsets) {
    pdl_wait();
    if (warp == 0) {      // the experts' row tiles, summed
      int before = 0;
      for (int e0 = 0; e0 < a.experts; e0 += 32) {
        const int e = e0 + lane, begin = e < a.experts ? bs_offset(a.offsets, e, a.M) : 0;
        int sum = e < a.experts ? (max(0, bs_offset(a.offsets, e + 1, a.M) - begin) + NT - 1) / NT : 0;
        if (e < a.experts) first_row[e] = begin;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += up;
        }
        if (e < a.experts) tiles_before[e + 1] = before + sum;
        before += __shfl_sync(0xffffffffu, sum, 31);
      }
      if (lane == 0) tiles_before[0] = 0, first_row[a.experts] = bs_offset(a.offsets, a.experts, a.M);
    }
  }
  pdl_trigger();
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot_ptr, 0);
  if (splits > 1) cluster_sync_all();             // every block of the cluster runs and has its barriers

  const int f_tiles = (a.N + 127) >> 7;
  const int row_tiles = a.offsets ? tiles_before[a.experts] : (a.M + NT - 1) / NT;
  const int num_tiles = row_tiles * f_tiles;
  auto tile_of = [&](int t) {                     // (feature tiles run fastest: blocks that run together read the same rows)
    const int row_tile = row_tiles == 1 ? 0 : t / f_tiles;
    BsTile m;
    int begin = 0, n = a.M, tiles = row_tiles, j = row_tile;
    m.expert = 0;
    if (a.offsets) {
      int lo = 0, hi = a.experts;                 // tiles_before[lo] <= row_tile < tiles_before[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tiles_before[mid] <= row_tile) lo = mid; else hi = mid;
      }
      begin = first_row[lo];
      n = first_row[lo + 1] - begin;
      tiles = tiles_before[lo + 1] - tiles_before[lo];
      j = row_tile - tiles_before[lo];
      m.expert = lo;
    }
    const int per = ((n + tiles - 1) / tiles + 15) & ~15;      // equal tiles (at most NT rows, and the last is not empty)
    m.first = begin + j * per;
    m.rows = min(per, n - j * per);
    m.feature = (t - row_tile * f_tiles) << 7;
    return m;
  };
  auto w_row = [&](const BsTile& m, int kb) { return ((m.expert * f_tiles + (m.feature >> 7)) * a.runs + kb) << 7; };      // of the tile's block in the matrix of blocks

  auto source = [&](const BsTile& m, int r) {     // the row of x that the tile's row r is
    const int at = m.first + min(r, m.rows - 1);
    return a.offsets && (a.modes & kBsByPair) ? min(bs_pair(a.order, at, a.M) / a.top, a.x_rows - 1) : at;
  };

  if (warp == 0) {
    const uint32_t leader = umma_leader();
    int ahead = 0, it = 0, s = 0;
    uint32_t phase = 1;
    bool ok = true;
    auto bytes = [&](const BsTile& m) { return kBsWBytes + (kCodes ? ((m.rows + 31) >> 5) * 32 * kBlk : 0); };
    if (!a.offsets) {
      for (int t = cluster_id; t < num_tiles && ahead < a.stages; t += clusters) {
        const BsTile m = tile_of(t);
        for (int kb = kb0; kb < kb1 && ahead < a.stages; ++kb, ++ahead)
          if (leader) {
            mbar_expect_tx(full_bar(ahead), bytes(m));
            tma_load_2d(base + ahead * S::kStage, &map_w, 0, w_row(m, kb), full_bar(ahead));
          }
      }
      pdl_wait();
    }
    for (int t = cluster_id; t < num_tiles && ok; t += clusters) {
      const BsTile m = tile_of(t);
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t stage = base + s * S::kStage;
        if (it >= ahead) {
          if (!mbar_wait_warp(empty_bar(s), phase)) {
            if (a.error_word && leader) atomicExch(a.error_word, 0x7C00C1);
            ok = false;
            break;
          }
          if (leader) {
            mbar_expect_tx(full_bar(s), bytes(m));
            tma_load_2d(stage, &map_w, 0, w_row(m, kb), full_bar(s));
          }
          __syncwarp();
        }
        if constexpr (kCodes) {
          if (leader) {
#pragma unroll
            for (int i = 0; i < NT / 32; ++i)     // (the last box may reach into the next tile's rows, or past the last: such columns are never stored)
              if (32 * i < m.rows) tma_load_2d(stage + kBsWBytes + i * 32 * kBlk, &map_x, kb * kBlk, m.first + 32 * i, full_bar(s));
          }
          __syncwarp();
        }
        if (++s == a.stages) { s = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = umma_leader();
    if (!a.offsets) pdl_wait();                   // (the bounded waits begin when the kernel before is over)
    int s = 0, b = 0;
    uint32_t phase = 0, acc_phase = 1;
    bool ok = true;
    for (int t = cluster_id; t < num_tiles && ok; t += clusters) {
      const BsTile m = tile_of(t);
      // D fp32, A and B e4m3, both K-major, N = the rows, M = 128
      const uint32_t idesc = (1u << 4) | ((uint32_t)((m.rows + 15) >> 4) << 18) | ((128u >> 4) << 24);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_warp(acc_empty_bar(b), acc_phase)) {
          if (a.error_word && leader) atomicExch(a.error_word, 0x7C00C4);
          ok = false;
          break;
        }
        if (!mbar_wait_warp(full_bar(s), phase)) {
          if (a.error_word && leader) atomicExch(a.error_word, 0x7C00C2);
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        const uint32_t w_src = umma_low_k128(base + s * S::kStage), x_src = w_src + (kBsWBytes >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f8_warp(leader, tmem_base + b * NT, w_src + 2 * k, x_src + 2 * k, idesc, k != 0);
        if (leader) {
          umma_commit(acc_full_bar(b));
          umma_commit(empty_bar(s));
        }
        __syncwarp();
        if (++s == a.stages) { s = 0; phase ^= 1; }
        if (++b == S::kBufs) { b = 0; acc_phase ^= 1; }
      }
    }
  } else if (warp < 2 + S::kStorers) {
    const int quarter = warp & 3, c0 = ((warp - 2) >> 2) * S::kCols;
    const int et = threadIdx.x - 64, lane8 = lane >> 2, pair = (lane & 3) * 2;
    int slot = 0, b = 0;
    uint32_t slot_phase = 0, acc_phase = 0;
    bool ok = true;
    if (!a.offsets) pdl_wait();                   // (y may be memory that the kernel before still reads)
    for (int t = cluster_id; t < num_tiles; t += clusters) {
      const BsTile m = tile_of(t);
      // sums of features quarter * 32 + 16 h + lane8 + 8 i, columns c0 + 8 j + pair and the next: [h][2 j + i]
      f32x2 sum[2][S::kCols / 4];
#pragma unroll
      for (int c = 0; c < S::kCols / 4; ++c) sum[0][c] = sum[1][c] = f2_pack(0.f, 0.f);
      f32x2 scale[S::kCols / 8];
      auto wait_scales = [&]() {
        if (ok && !mbar_wait_warp(scale_full_bar(slot), slot_phase)) {
          if (a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00C7);
          ok = false;
        }
      };
      auto read_scales = [&]() {
        const float* from = step_scales + slot * S::kScales + (lane8 & 1) * (NT + 8) + c0 + pair;
#pragma unroll
        for (int j = 0; j < S::kCols / 8; ++j) scale[j] = *reinterpret_cast<const f32x2*>(from + 8 * j);
      };
      for (int kb = kb0; kb < kb1; ++kb) {
        const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + b * NT + c0;
        uint32_t v[2][S::kCols / 2];
        auto add = [&](int h) {
#pragma unroll
          for (int j = 0; j < S::kCols / 8; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              sum[h][2 * j + i] = f2_fma(f2_pack(__uint_as_float(v[h][4 * j + 2 * i]), __uint_as_float(v[h][4 * j + 2 * i + 1])), scale[j], sum[h][2 * j + i]);
        };
        // What bounds tiles of up to 64 rows is this loop's latency: both loads are on their way while the scales are waited for and read (of 32 and 64
        // rows, 112 steps: 38.2 and 37.3 us; waited for ahead of one load after the other 38.8 and 42.0).  Of 128 rows it is shared memory, and the first
        // load's sums are added under the second (55.3 us, 67.0 the other way).
        if constexpr (NT >= 128) wait_scales();
        if (ok && !mbar_wait_warp(acc_full_bar(b), acc_phase)) {
          if (a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00C3);
          ok = false;
        }
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        tmem_ld_16x256b<S::kCols>(acc, v[0]);
        if constexpr (NT >= 128) {
          read_scales();
          asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
          tmem_ld_16x256b<S::kCols>(acc + (16u << 16), v[1]);
          add(0);
        } else {
          tmem_ld_16x256b<S::kCols>(acc + (16u << 16), v[1]);
          wait_scales();
          read_scales();
        }
        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(acc_empty_bar(b));
          if ((slot & 3) == 3) mbar_arrive(scale_empty_bar(slot));      // (this step's scales have been read, and those of the three before)
        }
        if constexpr (NT < 128) add(0);
        add(1);
        if (++slot == kBsSlots) { slot = 0; slot_phase ^= 1; }
        if (++b == S::kBufs) { b = 0; acc_phase ^= 1; }
      }
      // The sums cross shared memory, column by column, where a rolled loop finishes them, eight outputs of a column a thread (unrolled over a
      // thread's own sums, the activations' code would be fetched anew for every tile).  Block r of a cluster finishes features r * per .. of the tile.
      const int log_splits = 31 - __clz(splits), per = 128 >> log_splits, stride = per + 4;
      asm volatile("bar.sync 1, %0;\n" ::"r"(32 * S::kStorers) : "memory");       // (the last tile's sums have been read)
      if (splits == 1) {
        float* dst = red + (c0 + pair) * 132 + quarter * 32 + lane8;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < S::kCols / 4; ++q) {
            float* at = dst + (q >> 1) * 8 * 132 + 16 * h + 8 * (q & 1);
            f2_unpack(sum[h][q], at[0], at[132]);
          }
        asm volatile("bar.sync 1, %0;\n" ::"r"(32 * S::kStorers) : "memory");
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int feature = quarter * 32 + 16 * h + 8 * i + lane8;
            const int owner = feature >> (7 - log_splits);
            const uint32_t dst = map_to_cta(smem_u32(red + (rank * NT + c0 + pair) * stride + (feature & (per - 1))), owner);
            const uint32_t bar = map_to_cta(red_bar, owner);
#pragma unroll
            for (int j = 0; j < S::kCols / 8; ++j) {
              float lo, hi;
              f2_unpack(sum[h][2 * j + i], lo, hi);
              st_async_f32(dst + 8 * j * stride * 4, lo, bar);
              st_async_f32(dst + (8 * j + 1) * stride * 4, hi, bar);
            }
          }
        if (et == 0) mbar_expect_tx(red_bar, 128 * NT * 4);      // (the stores themselves count on the owner's barrier: no fence, no arrivals)
        if (!mbar_wait_cluster(red_bar, 0)) {
          if (a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00C5);
          ok = false;
        }
      }
      if (!ok) continue;
      switch (a.act) {
        case MOE_ACT_NONE: bs_finish<MOE_ACT_NONE, NT>(red, log_splits, rank, m, a, y, ldy, et, 32 * S::kStorers); break;
        case MOE_ACT_RELU2: bs_finish<MOE_ACT_RELU2, NT>(red, log_splits, rank, m, a, y, ldy, et, 32 * S::kStorers); break;
        case MOE_ACT_SILU: bs_finish<MOE_ACT_SILU, NT>(red, log_splits, rank, m, a, y, ldy, et, 32 * S::kStorers); break;
        case MOE_ACT_GELU: bs_finish<MOE_ACT_GELU, NT>(red, log_splits, rank, m, a, y, ldy, et, 32 * S::kStorers); break;
        case MOE_ACT_GLU_CLAMP: bs_finish<MOE_ACT_GLU_CLAMP, NT>(red, log_splits, rank, m, a, y, ldy, et, 32 * S::kStorers); break;
        default: bs_finish<MOE_ACT_SWIGLU, NT>(red, log_splits, rank, m, a, y, ldy, et, 32 * S::kStorers); break;
      }
    }
  } else {
    // this helper's steps: the first, and every kHelpers-th after it
    const int helper = warp - 2 - S::kStorers;
    int kb = kb0 + helper, step = helper, s = helper % a.stages, slot = helper;      // (step: counted over all tiles)
    uint32_t phase = 1 ^ ((helper / a.stages) & 1), slot_phase = 1;
    bool ok = true, waited = a.offsets != nullptr, outside = false;
    auto advance = [&]() {
      kb += S::kHelpers;
      step += S::kHelpers;
      for (s += S::kHelpers; s >= a.stages; s -= a.stages) phase ^= 1;
      if ((slot += S::kHelpers) >= kBsSlots) { slot -= kBsSlots; slot_phase ^= 1; }
    };
    for (int t = cluster_id; t < num_tiles && ok; t += clusters, kb -= kb1 - kb0) {
      const BsTile m = tile_of(t);
      const float* ws = a.w_scales + ((size_t)m.expert * a.scale_rows + bs_scale_row(m.feature, a.pairs)) * a.runs;
      if constexpr (kCodes) {
        if (!waited) pdl_wait();
        waited = true;
        // (four of this helper's steps at a time: their loads are on their way together)
        while (kb < kb1 && ok) {
          float v[4][NT / 32], even[4], odd[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = min(kb + j * S::kHelpers, kb1 - 1);
            even[j] = ws[at];
            odd[j] = a.pairs ? ws[a.runs + at] : even[j];
#pragma unroll
            for (int i = 0; i < NT / 32; ++i) v[j][i] = a.x_scales[(size_t)at * a.lds + m.first + min(lane + 32 * i, m.rows - 1)];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (kb >= kb1) break;
            if (!mbar_wait_warp(scale_empty_bar(slot), slot_phase)) {
              ok = false;
              break;
            }
            float* scales = step_scales + slot * S::kScales;
#pragma unroll
            for (int i = 0; i < NT / 32; ++i) {
              outside |= a.outside(v[j][i]);
              scales[lane + 32 * i] = v[j][i] * even[j];
              scales[NT + 8 + lane + 32 * i] = v[j][i] * odd[j];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(scale_full_bar(slot));
            advance();
          }
        }
      } else {
        // Eight lanes a row, sixteen columns each; two rows a lane at a time (`turn`: rows 8 half + sub and the fourth after it), the next two (of this
        // step or this helper's next) on their way.  What the first MMA waits for is this warp's instructions between the kernel before and the first
        // codes, one behind the other: all that does not need x is done ahead of them.
        static_assert(NT == 16, "two halves of eight rows");
        const TX* x = reinterpret_cast<const TX*>(a.x);
        const int sub = lane >> 3, eighth = lane & 7;
        const TX* row[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) row[i] = x + (size_t)source(m, 4 * i + sub) * a.ldx + eighth * 16;
        struct Rows { uint4 raw[2][sizeof(TX)]; float even, odd; };
        auto ask = [&](Rows& q, int run, bool half) {
          if (run >= kb1) return;
          const bool whole = a.vec && (run + 1) * kBlk <= a.K;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const TX* p = (half ? row[2 + h] : row[h]) + run * kBlk;
            const bool in = (half ? 8 : 0) + 4 * h + sub < m.rows;
            if (whole) {
#pragma unroll
              for (int i = 0; i < (int)sizeof(TX); ++i) q.raw[h][i] = in ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
            } else bs_ask16<TX, false>(p, in ? a.K - run * kBlk - eighth * 16 : 0, q.raw[h]);
          }
          q.even = ws[run];
          q.odd = a.pairs ? ws[a.runs + run] : q.even;
        };
        bool half = false;
        auto turn = [&](Rows& now, Rows& next) {
          const bool last = half || m.rows <= 8;
          ask(next, last ? kb + S::kHelpers : kb, !last);
          if (!half && ((step >= a.stages && !mbar_wait_warp(empty_bar(s), phase)) || (step >= kBsSlots && !mbar_wait_warp(scale_empty_bar(slot), slot_phase)))) {
            ok = false;
            return;
          }
          float* scales = step_scales + slot * S::kScales;
          unsigned char* codes = smem_gen + s * S::kStage + kBsWBytes;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = (half ? 8 : 0) + 4 * h + sub;
            uint32_t largest = bs_largest16<TX>(now.raw[h]);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
            float scale, inverse;
            bs_run_scale(largest, scale, inverse);
            outside |= a.outside(scale);
            if (r < m.rows) {
              *reinterpret_cast<uint4*>(codes + r * kBlk + ((eighth ^ (r & 7)) << 4)) = bs_codes16<TX>(now.raw[h], inverse);
              if (eighth == 0) {
                scales[r] = scale * now.even;
                scales[NT + 8 + r] = scale * now.odd;
              }
            }
          }
          if (last) {
            bs_fence_async_shared();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(scale_full_bar(slot));
              mbar_arrive(full_bar(s));
            }
            advance();
          }
          half = !last;
        };
        Rows p, q;
        if (!waited) pdl_wait();
        waited = true;
        ask(p, kb, false);
        while (kb < kb1 && ok) {
          turn(p, q);
          if (kb < kb1 && ok) turn(q, p);
          else break;
        }
      }
      if (!ok && a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00C6);
    }
    if (outside)      // (any block of the cluster finishes outputs of these rows)
      for (int r = 0; r < splits; ++r) st_cluster_u32(map_to_cta(far_seen, r), 1u);
  }
  __syncwarp();
  if (splits > 1) {
    cluster_sync_all();                           // every block has sent its sums, also one that gave up waiting for others',
    if (warp == 0) mbar_wait_warp(red_bar, 0);    // and none leaves before what was sent to it has come
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(S::kTmemCols) : "memory");
  }
  // Rows with far scales: by the producer's warp, whose instructions here delay no other.
  if (warp == 0 && *reinterpret_cast<volatile uint32_t*>(smem_gen + (far_seen - base)))
    for (int t = cluster_id; t < num_tiles; t += clusters) bs_tile_apart<TX, TO>(a, tile_of(t), rank, splits, lane, y, ldy);
}

template <int NT>
static constexpr uint32_t bs_smem(int stages, int splits, int experts) {
  using S = BsShape<NT, true>;
  return 1024u + stages * S::kStage + kBsBarBytes + 4 * (kBsSlots * S::kScales + bs_red_floats<NT>(splits) + 2 * (experts + 1));
}

// The blocks that share a tile's runs: 8, 4 or 2 where there is room for them beside the other tiles' and the runs are enough to pay for the exchange.
// (us by 1 / 2 / 4 / 8 blocks a tile: 8 rows 4,096 -> 4,096 14.2 / 9.8 / 8.3 / 9.0, 14,336 -> 4,096 43 / 25 / 16.7 / 15.0, 4,096 -> 6,144 14.2 / 10.6 /
// 9.1 / 14.8, 2,048 -> 2,048 8.2 / 6.5 / 5.9 / 6.1; 4 rows 512 -> 1,024 4.0 / 4.5 / 4.3; 20 rows 512 -> 1,024 5.5 / 6.3 / 5.9.  By 4 / 8 about the 64 runs from which
// it is 8, at 32, 40, 48, 56, 64, 80 runs: 8 rows and 4,096 features 7.8 / 8.1, 8.4 / 8.9, 9.2 / 9.4, 9.8 / 9.8, 10.6 / 10.3, 12.1 / 11.6; 2,048 features 7.0 / 6.1,
// 7.6 / 6.8, 8.4 / 7.2, 9.0 / 7.5, 9.7 / 8.0, 11.0 / 8.7; 20 rows and 2,048 features 8.7 / 9.7, 9.5 / 10.5, 10.1 / 11.0, 10.7 / 11.4, 11.2 / 12.0, 12.4 / 12.6.)
static int bs_splits(int64_t tiles, int runs, int blocks) {
  if (tiles * 8 <= blocks && runs >= 64) return 8;
  if (tiles * 4 <= blocks && runs >= 8) return 4;
  return tiles * 2 <= blocks && runs >= 8 ? 2 : 1;
}
// Rows of a tile of codes: the fewest that give no more tiles than SMs; of a long matrix (64 runs) not fewer than 64 while there are that many rows, as every row tile
// reads the weights again.  (us in tiles of 32 / 64 / 128 rows: 333 rows 1,000 -> 1,302 8.2 / 9.5 / 11.4, 128 rows 4,096 -> 4,096 13.7 / 14.1 / 15.6, 256 rows
// 18.0 / 16.7 / 20.0, 100 rows 2,048 -> 2,048 8.9 / 10.2 / 11.8, 64 rows 14,336 -> 4,096 19.2 / 18.1 / 25.5, 128 rows 28.1 / 26.1 / 26.3, 128 rows 4,096 ->
// 14,336 29.2 / 27.9 / 24.9.  32 / 64 about those 64 runs, at 32, 40, 48, 56, 64, 80 runs and 4,096 features: 64 rows 12.0 / 12.0, 13.1 / 12.5, 14.2 / 13.1, 15.3 / 13.7,
// 16.5 / 14.2, 18.9 / 15.9; 128 rows 14.8 / 13.8, 17.2 / 15.1, 19.4 / 16.3, 21.6 / 17.5, 23.5 / 18.6, 28.0 / 21.1.  Where eight blocks share a tile it is the other way:
// 64 rows and 2,048 features at 64 runs 11.8 / 19.9, which the rule does not know.)
static int bs_tile_rows(int rows, int features, int runs) {
  const int64_t f_tiles = ceil_div(features, 128);
  if (rows <= 32 || (ceil_div(rows, 32) * f_tiles <= 148 && runs < 64)) return 32;
  return rows <= 64 || ceil_div(rows, 64) * f_tiles <= 148 ? 64 : 128;
}

// How a product runs: blocks in the grid, those that share a tile, steps of a block at most, stages of its ring.
struct BsPlan { int grid, splits, steps, stages; };
template <int NT, bool CODES> static int bs_plan(int M, int N, int runs, int experts, BsPlan& p) {      // experts: 0 for one matrix
  using S = BsShape<NT, CODES>;
  constexpr int kBlocks = 148 * S::kPerSm;
  const int64_t row_tiles = experts ? M / NT + (M < experts ? M : experts) : ceil_div(M, NT), tiles = row_tiles * ceil_div(N, 128);
  // (a tile of 128 rows is never shared: bs_tile_rows takes such tiles where smaller ones are more than the SMs)
  p.splits = experts || NT >= 128 ? 1 : bs_splits(tiles, runs, CODES ? 148 : 296);
  if (tiles * p.splits > 0x7fffffff) return TIB_E_SIZE;
  p.grid = (int)(p.splits > 1 ? tiles * p.splits : tiles < kBlocks ? tiles : kBlocks);      // (a cluster has one tile: its sums' place is used once)
  const int64_t steps = (int64_t)ceil_div(runs, p.splits) * ceil_div64(tiles * p.splits, p.grid);
  p.steps = (int)(steps < 0x7fffffff ? steps : 0x7fffffff);
  p.stages = 1;
  while (p.stages < kBsMaxStages && p.stages < p.steps && bs_smem<NT>(p.stages + 1, p.splits, experts) <= (S::kPerSm > 1 ? 113u * 1024 : (uint32_t)kMostSmem)) ++p.stages;
  // (A wait by parity tells a stage's last use from the one before only while a helper's step before implies the latter is over: with no more helpers
  // than stages, or every stage used once.)
  return !CODES && p.stages < S::kHelpers && p.stages < p.steps ? TIB_E_SMEM : TIB_OK;
}
// Rows of a tile for rows given as codes.  (Of sorted rows tiles of 32 are ahead, or near, up to where pairs of SMs take over.  32 / 64 / 128 rows a tile, us: 25 rows
// an expert 19.5 / 18.5 / 24.3, 50 21.5 / 25.0 / 25.6, 87 30.7 / 33.1 / 35.5, 32 of 28 experts 17.4 / 20.0 / 23.6; with a skew 16.2 / 16.2 / 20.7.)
static int bs_code_rows(int M, int N, int runs, int experts) {
  return !experts ? bs_tile_rows(M, N, runs) : M < (int64_t)experts * 128 ? 32 : 128;
}

template <int NT, typename TX, typename TO>
static int launch_block_scaled(const CUtensorMap& map_w, const CUtensorMap& map_x, BsArgs& a, void* y, int64_t ldy, cudaStream_t stream) {
  constexpr bool kCodes = std::is_same_v<TX, uint8_t>;
  const int experts = a.offsets ? a.experts : 0;
  BsPlan plan;
  const int rc = bs_plan<NT, kCodes>(a.M, a.N, a.runs, experts, plan);
  if (rc != TIB_OK) return rc;
  a.stages = plan.stages;
  auto kern = block_scaled_tcgen05_kernel<NT, TX, TO>;
  static bool allowed[64];      // (by device: the attribute belongs to its context)
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && !(device < 64 && allowed[device])) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
  if (e != cudaSuccess) return (int)e;
  if (device < 64) allowed[device] = true;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(BsShape<NT, kCodes>::kThreads);
  cfg.dynamicSmemBytes = bs_smem<NT>(plan.stages, plan.splits, experts);
  cfg.stream = stream;
  cfg.gridDim = dim3((unsigned)plan.grid);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)plan.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // (see launch_dependent in common.cuh)
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent_launch_flag() ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, map_w, map_x, (const BsArgs)a, (TO*)y, ldy);
  if (e != cudaSuccess) return (int)e;
  TIB_LAUNCH_CHECK();
  return TIB_OK;
}

}  // namespace tib

using namespace tib;

// x_dtype TIB_BF16 or TIB_F32: rows [rows, K] (row stride ldx) that are quantised on the way, for each tile of 16 rows x
// 128 features; -1: codes
// [x_rows, runs * 128] and scales [runs, lds] as tib_quantize_rows leaves them, row m of them for row m of y.  w: codes in blocks
// [experts, ceil(N / 128), runs, 128, 128], features and columns behind the last zero, and scales [experts, scale_rows, runs] (`pairs`: of (gate, up) row pairs); y: [M, N] in y_dtype (row stride ldy), or [M, N / 2] of a gated activation.
// offsets [experts + 1] and order [M]: rows sorted by expert as tib_moe_expert_product takes them; offsets null: one matrix for all rows.  far_low, far_high:
// which rows' scales keep normal with every one of w's (BsFar).
TIB_API int tib_block_scaled_tcgen05(const void* x, int x_dtype, int64_t ldx, int x_rows, const float* x_scales, int64_t lds, const void* w,
                                     const float* w_scales, int scale_rows, int pairs, void* y, int y_dtype, int64_t ldy, int M, int N, int K,
                                     const int* offsets, const int* order, int experts, int top, int x_by_pair, int act, float limit,
                                     float alpha, const float* row_scale, float far_low, float far_high, int* error_word, cudaStream_t stream) {
  if (M == 0 || N == 0) return TIB_OK;
  const bool is_codes = x_dtype < 0;
  if (!x || !w || !w_scales || !y || M < 0 || N < 0 || K < 1 || experts < 1 || top < 1 || x_rows < 1) return TIB_E_ARG;
  if ((is_codes && (!x_scales || (offsets && x_by_pair) || x_rows < M || lds < M || lds > 0x7fffffff)) || (offsets && !order) || (row_scale && !order)) return TIB_E_ARG;
  if (act < MOE_ACT_NONE || act > MOE_ACT_GELU || (moe_act_gated(act) && !pairs) || (pairs && N % 2)) return TIB_E_SIZE;
  if (x_dtype > TIB_BF16 || (y_dtype != TIB_BF16 && y_dtype != TIB_F32)) return TIB_E_DTYPE;
  if (experts > kBsMaxExperts || (int64_t)experts * ceil_div(N, 128) * ceil_div(K, kBlk) > (0x7fffffff >> 7)) return TIB_E_SIZE;
  if ((((uintptr_t)w) & 15) || (is_codes && (((uintptr_t)x) & 15))) return TIB_E_ALIGN;
  BsArgs a;
  a.x = x; a.ldx = ldx; a.x_scales = x_scales; a.w = static_cast<const unsigned char*>(w); a.w_scales = w_scales; a.scale_rows = scale_rows; a.pairs = pairs;
  a.vec = !is_codes && ((uintptr_t)x & 15) == 0 && (ldx * (x_dtype == TIB_BF16 ? 2 : 4)) % 16 == 0;
  a.lds = (int)lds; a.M = M; a.N = N; a.K = K; a.runs = ceil_div(K, kBlk); a.x_rows = x_rows; a.offsets = offsets; a.order = order; a.experts = experts; a.top = top;
  const bool wide = ((uintptr_t)y & 15) == 0 && (ldy * (y_dtype == TIB_BF16 ? 2 : 4)) % 16 == 0;
  a.modes = (x_by_pair ? kBsByPair : 0) | (wide ? kBsWide : 0);
  a.far_low = far_low; a.far_high = far_high;
  a.act = act; a.limit = limit; a.alpha = alpha; a.row_scale = row_scale; a.error_word = error_word;
  CUtensorMap map_w, map_x;
  int rc = bs_make_map(&map_w, w, (int64_t)experts * ceil_div(N, 128) * a.runs * 128, kBlk, 128);
  if (rc != TIB_OK) return rc;
  map_x = map_w;
  if (is_codes) {
    rc = bs_make_map(&map_x, x, x_rows, (int64_t)a.runs * kBlk, 32);
    if (rc != TIB_OK) return rc;
  }
#define TIB_BS_GO(NT, TX)                                                                                                  \
  return y_dtype == TIB_BF16 ? launch_block_scaled<NT, TX, __nv_bfloat16>(map_w, map_x, a, y, ldy, stream)                 \
                             : launch_block_scaled<NT, TX, float>(map_w, map_x, a, y, ldy, stream)
  if (is_codes) {
    const int nt = bs_code_rows(M, N, a.runs, offsets ? experts : 0);
    if (nt == 32) TIB_BS_GO(32, uint8_t);
    if (nt == 64) TIB_BS_GO(64, uint8_t);
    TIB_BS_GO(128, uint8_t);
  }
  if (x_dtype == TIB_BF16) TIB_BS_GO(16, __nv_bfloat16);
  TIB_BS_GO(16, float);
#undef TIB_BS_GO
}

// How a product of M rows (codes, or not) with one matrix (experts 0) or sorted by expert runs here: {rows of a tile at most, blocks that share a tile, steps of a
// block at most, stages of its ring}.
TIB_API int tib_block_scaled_tcgen05_plan(int codes, int M, int N, int K, int experts, int* plan) {
  if (!plan || M < 1 || N < 1 || K < 1 || experts < 0 || experts > kBsMaxExperts) return TIB_E_ARG;
  const int runs = ceil_div(K, kBlk), nt = codes ? bs_code_rows(M, N, runs, experts) : 16;
  BsPlan p;
  const int rc = nt == 16 ? bs_plan<16, false>(M, N, runs, experts, p) : nt == 32 ? bs_plan<32, true>(M, N, runs, experts, p)
               : nt == 64 ? bs_plan<64, true>(M, N, runs, experts, p) : bs_plan<128, true>(M, N, runs, experts, p);
  plan[0] = nt; plan[1] = p.splits; plan[2] = p.steps; plan[3] = p.stages;
  return rc;
}
