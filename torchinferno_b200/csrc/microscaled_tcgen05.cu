// Products of 4-bit microscaled operands on the 5th-generation tensor cores, for few rows and for rows sorted by expert:
//     y[m, n] = act(r[m] f[n] (sum over runs b of s[m, b] S[n, b] (sum over the 16 columns of run b of x[m, k] w[n, k])))
//
// The weights are the 128-row operand of the MMA and the rows its N dimension: a tile is 128 features x up to NT rows, the rows rounded up to 16
// only, and the accumulator, which stays in tensor memory for the whole sum, is the transposed output (TMEM lane = feature, column = row).  A step of the loop
// is 256 columns: the 128-byte row of the swizzle, eight copies of scales (512 bytes each) to tensor memory, four MMAs.  The scales of a stage of the
// ring have columns of their own, so that they are free when the stage is.
//   warp 0       producer: four copies a step, each of bytes that lie side by side: 16 KB of codes of w, 2 KB of its scales, the rows' codes and scales
//   warp 1       copies scales and issues tcgen05.mma; owns the TMEM allocation
//   the next 4 or 8   epilogue: some rows at a time, a lane a feature, so that a warp writes 32 outputs of a row side by side; two accumulators take turns.  Of up to eight short
//                rows (ms_makes_rows) they first make the codes, straight into the ring, where no kernel has made them before
// A matrix of few tiles is split by steps over a cluster of up to eight blocks, whose sums meet in distributed shared memory, added in the order of the
// steps.
// What bounds it, at few rows: memory.  8 rows 4,096 -> 28,672: 12.3 us for 66 MB (5.4 TB/s, 84 % of the measured copy bandwidth; without the copies 7.1); 14,336 -> 4,096 9.2 us
// for 33 MB, 4,096 -> 4,096 5.1 us for 9.4 MB, of which some 3.5 are the start, the exchange and the end.  With the kernel that makes the rows' codes ahead of it, whose time
// the first copies of weights fill, 14.5, 10.3 and 6.4 us.  In tiles of 128 rows the finishing of 128 x 128 outputs: 128 rows 4,096 -> 28,672 16.8 us with eight warps that
// have their next columns on their way, 22.5 with four that wait for each eight of them, 12.8 without; and their number: 224 tiles are a round of 148 SMs and one half
// empty.  Every wait is bounded and reports in error_word.
#include "microscaled.cuh"

namespace tib {

constexpr int kMtMaxExperts = 1024, kMtMaxStages = 8;
constexpr uint32_t kMtWBytes = kMsTileRows * kMsStepBytes, kMtBarBytes = 256;

template <int NT> struct MtShape {
  static constexpr int kPerSm = NT <= 32 ? 2 : 1;                                // blocks of an SM
  static constexpr int kStorers = NT >= 128 ? 8 : 4, kThreads = 64 + 32 * kStorers, kCols = NT / (kStorers / 4);      // (columns of a storer)
  static constexpr int kTurn = NT >= 128 ? 16 : 8;                               // columns that it takes at a time
  // Tensor memory: accumulators (two; one of a shared tile, which is a block's only one), then 32 columns of scales a stage.  At most:
  static constexpr uint32_t tmem_cols(int splits) { return (splits > 1 ? 256 : 512) / kPerSm; }
  __host__ __device__ static constexpr uint32_t scale_cols(int splits) { return splits > 1 ? NT : 2 * NT; }
  static constexpr int stages(int splits) { return (tmem_cols(splits) - scale_cols(splits)) / 32 < kMtMaxStages ? (tmem_cols(splits) - scale_cols(splits)) / 32 : kMtMaxStages; }
  static constexpr uint32_t kStage = kMtWBytes + NT * kMsStepBytes + 2 * kMsStepScales;
};
// of the sums of a shared tile: (a column's 128 / splits sums and four more, so that those that a warp writes at a time fall on all banks)
template <int NT> __host__ __device__ constexpr int mt_red_floats(int splits) { return splits > 1 ? NT * (128 + 4 * splits) : 0; }

// (the binary logarithm of) how many of eight loads are of the same of M rows.
__host__ __device__ constexpr int mt_more_loads(int M) { return M > 4 ? 0 : M > 2 ? 1 : 4 - M; }

struct MtTile { int expert, first, rows, group, scale_tile, feature; };

// An output (of a gated unit: from its gate g and up u).
template <int ACT> __device__ __forceinline__ float mt_act(float g, float u, const MsArgs& a) {
  if constexpr (moe_act_gated(ACT)) return bs_gated<ACT>(g, u, a.limit, a.alpha);
  else return bs_act<ACT>(g);
}

// MAKE: up to eight rows, short ones, whose codes the finishing warps, idle till then, put into the ring themselves: a thread a run of a step.  Every block looks for the rows' largest
// numbers first.
template <int NT, int ACT, typename TO, bool MAKE>
__global__ void __launch_bounds__(MtShape<NT>::kThreads, MtShape<NT>::kPerSm)
microscaled_tcgen05_kernel(const __grid_constant__ MsArgs a, TO* __restrict__ y, int64_t ldy) {
  using S = MtShape<NT>;
  constexpr int kGated = moe_act_gated(ACT) ? 1 : 0;
  const int splits = (int)cluster_size(), rank = (int)cluster_rank();
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem_gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + a.stages * S::kStage;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kMtMaxStages + s); };
  auto acc_full_bar = [&](int b) { return bars + 8u * (2 * kMtMaxStages + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * kMtMaxStages + 2 + b); };
  const uint32_t red_bar = bars + 8u * (2 * kMtMaxStages + 4), tmem_slot = red_bar + 8;
  static_assert(8 * (2 * kMtMaxStages + 5) + 8 <= kMtBarBytes, "the barriers' share of shared memory");
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_gen + (tmem_slot - base));
  float* red = reinterpret_cast<float*>(smem_gen + (bars - base) + kMtBarBytes);         // [splits][NT][128 / splits + 4] sums
  float* tile_factors = red + mt_red_floats<NT>(splits);                                 // [2][NT][2] what a row's sums are multiplied by (ms_row_scales), of two tiles in turn
  int* tiles_before = reinterpret_cast<int*>(tile_factors + 4 * NT);                     // [experts + 1] where rows are sorted, and
  int* first_row = tiles_before + a.experts + 1;                                         // [experts + 1] their offsets

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int cluster_id = blockIdx.x / splits, clusters = gridDim.x / splits;
  const int step0 = (int)((int64_t)a.steps * rank / splits), step1 = (int)((int64_t)a.steps * (rank + 1) / splits);
  if (warp == 0) {
    if (lane < a.stages) {
      mbar_init(full_bar(lane), MAKE ? 1 + S::kStorers : 1);
      mbar_init(empty_bar(lane), 1);
    }
    if (lane < 2) {
      mbar_init(acc_full_bar(lane), 1);
      mbar_init(acc_empty_bar(lane), S::kStorers);
    }
    if (lane == 0) mbar_init(red_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tmem_slot), "r"(a.tmem_cols) : "memory");
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
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  pdl_trigger();      // (tensor memory is this block's by now: a block of the kernel behind it cannot take it first)
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot_ptr, 0);
  if (splits > 1) cluster_sync_all();             // every block of the cluster runs and has its barriers

  const int f_tiles = (a.N + 127) >> 7;
  const int row_tiles = a.offsets ? tiles_before[a.experts] : (a.M + NT - 1) / NT;
  const int num_tiles = row_tiles * f_tiles;
  auto tile_of = [&](int t) {                     // (feature tiles run fastest: blocks that run together read the same rows)
    const int row_tile = row_tiles == 1 ? 0 : t / f_tiles;
    MtTile m;
    int begin = 0, n = a.M, j = row_tile;
    m.expert = 0;
    m.scale_tile = m.group = 0;
    if (a.offsets) {
      int lo = 0, hi = a.experts;                 // tiles_before[lo] <= row_tile < tiles_before[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tiles_before[mid] <= row_tile) lo = mid; else hi = mid;
      }
      begin = first_row[lo];
      n = first_row[lo + 1] - begin;
      j = row_tile - tiles_before[lo];
      m.expert = lo;
      m.scale_tile = ms_first_tile(begin, lo);
      m.group = ms_first_group(begin, lo);
    }
    m.first = begin + j * NT;
    m.rows = min(NT, n - j * NT);
    m.group += j * (NT / kMsGroup);
    m.scale_tile += j * NT >> 7;                  // (tiles of fewer than 128 rows: the launch sees to it that there is one)
    m.feature = (t - row_tile * f_tiles) << 7;
    return m;
  };

  if (warp == 0) {
    const uint32_t leader = umma_leader();
    int ahead = 0, it = 0, s = 0;
    uint32_t phase = 1;
    bool ok = true;
    auto rows_bytes = [&](const MtTile& m) { return (uint32_t)((m.rows + kMsGroup - 1) / kMsGroup) * kMsGroupBytes; };
    auto ask_w = [&](const MtTile& m, int step, int s) {
      const uint32_t stage = base + s * S::kStage;
      const int block = (m.expert * f_tiles + (m.feature >> 7)) * a.steps + step;
      mbar_expect_tx(full_bar(s), MAKE ? kMtWBytes + kMsStepScales : kMtWBytes + 2 * kMsStepScales + rows_bytes(m));
      ms_bulk_load(stage, a.w + (size_t)block * kMtWBytes, kMtWBytes, full_bar(s));
      ms_bulk_load(stage + kMtWBytes + NT * kMsStepBytes, a.w_scales + (size_t)block * kMsStepScales, kMsStepScales, full_bar(s));
    };
    if (!a.offsets) {
      for (int t = cluster_id; t < num_tiles && ahead < a.stages; t += clusters) {
        const MtTile m = tile_of(t);
        for (int step = step0; step < step1 && ahead < a.stages; ++step, ++ahead)
          if (leader) ask_w(m, step, ahead);
      }
      pdl_wait();
    }
    for (int t = cluster_id; t < num_tiles && ok; t += clusters) {
      const MtTile m = tile_of(t);
      for (int step = step0; step < step1; ++step, ++it) {
        if (it >= ahead) {
          if (!mbar_wait_warp(empty_bar(s), phase)) {
            if (a.error_word && leader) atomicExch(a.error_word, 0x7C00E1);
            ok = false;
            break;
          }
          if (leader) ask_w(m, step, s);
          __syncwarp();
        }
        if (!MAKE && leader) {
          const uint32_t rows_at = base + s * S::kStage + kMtWBytes;
          ms_bulk_load(rows_at, a.x.codes + ((size_t)step * a.x.groups + m.group) * kMsGroupBytes, rows_bytes(m), full_bar(s));
          ms_bulk_load(rows_at + NT * kMsStepBytes + kMsStepScales, a.x.scales + ((size_t)m.scale_tile * a.steps + step) * kMsStepScales, kMsStepScales, full_bar(s));
        }
        __syncwarp();
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
      const MtTile m = tile_of(t);
      const uint32_t idesc = kMsIdesc | ((uint32_t)((m.rows + 15) >> 4) << 18) | ((128u >> 4) << 24);
      if (!mbar_wait_warp(acc_empty_bar(b), acc_phase)) {
        if (a.error_word && leader) atomicExch(a.error_word, 0x7C00E4);
        break;
      }
      for (int step = step0; step < step1; ++step) {
        if (!mbar_wait_warp(full_bar(s), phase)) {
          if (a.error_word && leader) atomicExch(a.error_word, 0x7C00E2);
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        const uint32_t stage = base + s * S::kStage, scales = stage + kMtWBytes + NT * kMsStepBytes;
        const uint32_t w_src = umma_low_k128(stage), x_src = w_src + (kMtWBytes >> 4), columns = tmem_base + S::scale_cols(splits) + 32 * s;
        if (leader) {
#pragma unroll
          for (int k = 0; k < 8; ++k) ms_copy_scales<1>(columns + 4 * k, scales + kMsChunkBytes * k);      // (four of w, four of the rows)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            ms_umma<1>(tmem_base + b * NT, w_src + 2 * k, x_src + 2 * k, idesc, columns + 4 * k, columns + 16 + 4 * k, step != step0 || k != 0);
          umma_commit(empty_bar(s));
        }
        __syncwarp();
        if (++s == a.stages) { s = 0; phase ^= 1; }
      }
      if (leader) umma_commit(acc_full_bar(b));
      __syncwarp();
      if (++b == 2) { b = 0; acc_phase ^= 1; }
    }
  } else {
    const int quarter = warp & 3, et = threadIdx.x - 64, c0 = ((warp - 2) >> 2) * S::kCols;
    int b = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    if (!a.offsets) pdl_wait();                   // (y may be memory that the kernel before still reads)
    const int own_row = et >> 4, own_run = et & 15;      // (of a step of eight rows)
    float r = 1.f, inverse = 1.f;
    int ring = 0;
    uint32_t ring_phase = 1;
    if constexpr (MAKE) {
      static_assert(NT == 32 && S::kStorers == 4, "eight rows of 16 runs are a thread's each");
      uint32_t* found = reinterpret_cast<uint32_t*>(tile_factors) + 32;      // [4 warps][8] (behind the eight rows' factors)
      // Eight loads of eight numbers a thread, all on their way at once; of fewer rows several of a row: load i is of row i >> more.
      const int more = mt_more_loads(a.M), mask = (1 << more) - 1;
      uint4 raw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i >> more, at = (et + (i & mask) * 128) * 8;
        raw[i] = row < a.M && at < a.K ? *reinterpret_cast<const uint4*>(a.made + row * a.ld_made + at) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t two = __vmaxu2(__vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu), __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu));
        const uint32_t most = __reduce_max_sync(0xffffffffu, max(two << 16, two & 0xffff0000u));
        if (lane == 0) found[(warp - 2) * 8 + i] = most;
      }
      asm volatile("bar.sync 1, %0;\n" ::"r"(32 * S::kStorers) : "memory");
      if (own_row < a.M) {
        uint32_t most = 0;
        for (int i = own_row << more; i <= (own_row << more | mask); ++i) most = max(most, max(max(found[i], found[8 + i]), max(found[16 + i], found[24 + i])));
        ms_row_scale(most, r, inverse);
      }
    }
    for (int t = cluster_id; t < num_tiles; t += clusters) {
      const MtTile m = tile_of(t);
      const int feature = m.feature + quarter * 32 + lane, n_out = a.N >> kGated;
      const float factor = a.w_factors[(size_t)m.expert * a.N + min(feature, a.N - 1)];
      float2* factors = reinterpret_cast<float2*>(tile_factors) + b * NT;
      if constexpr (MAKE) {
        if (own_run == 0 && own_row < m.rows) factors[own_row] = make_float2(r, 1.f);
      } else if (et < m.rows) {
        factors[et] = make_float2(a.x.factors[m.first + et], 1.f);
        if (a.row_scale) factors[et] = ms_row_scales(a.x.factors[m.first + et], a.row_scale[bs_pair(a.order, m.first + et, a.M)]);
      }
      asm volatile("bar.sync 1, %0;\n" ::"r"(32 * S::kStorers) : "memory");      // (the last tile but one is finished: its factors have been read)
      if constexpr (MAKE) {
        const __nv_bfloat16* src = a.made + own_row * a.ld_made;
        for (int step = step0; step < step1 && ok; ++step) {
          if (!mbar_wait_warp(empty_bar(ring), ring_phase)) {
            if (a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00E6);
            ok = false;
            break;
          }
          if (own_row < a.M) {
            const int run = step * (kMsStep / kMsRun) + own_run;
            unsigned char* rows_at = smem_gen + ring * S::kStage + kMtWBytes;
            uint4 raw[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              raw[i] = run * kMsRun + 8 * i < a.K ? *reinterpret_cast<const uint4*>(src + run * kMsRun + 8 * i) : make_uint4(0, 0, 0, 0);
            uint32_t scale;
            const uint2 codes = ms_run_codes<__nv_bfloat16>(raw, bs_largest16<__nv_bfloat16>(raw), inverse, scale);
            *reinterpret_cast<uint2*>(rows_at + ms_code_at(own_row, own_run * (kMsRun / 2))) = codes;
            rows_at[NT * kMsStepBytes + kMsStepScales + (own_run >> 2) * kMsChunkBytes + ms_scale_at(own_row) + (own_run & 3)] = (unsigned char)scale;
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(full_bar(ring));
          if (++ring == a.stages) { ring = 0; ring_phase ^= 1; }
        }
      }
      if (ok && !mbar_wait_warp(acc_full_bar(b), acc_phase)) {
        if (a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00E3);
        ok = false;
      }
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + b * NT;
      const int c1 = min(c0 + S::kCols, m.rows);
      // (a turn's columns are on their way while those before are finished)
      auto columns = [&](auto&& finish) {
        uint32_t v[2][S::kTurn];
        auto ask = [&](int i, int c) {
          if constexpr (S::kTurn == 16) tmem_ld16(acc + c, v[i]);
          else tmem_ld8(acc + c, v[i]);
        };
        if (c0 < c1) ask(0, c0);
#pragma unroll 1
        for (int c = c0; c < c1; c += 2 * S::kTurn) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (c + i * S::kTurn >= c1) break;
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
            if (c + (i + 1) * S::kTurn < c1) ask(i ^ 1, c + (i + 1) * S::kTurn);
            finish(c + i * S::kTurn, v[i]);
          }
        }
      };
      if (splits == 1)
        columns([&](int c, const uint32_t (&v)[S::kTurn]) {
          float s[S::kTurn];
#pragma unroll
          for (int j = 0; j < S::kTurn; ++j) {
            const float2 f = factors[min(c + j, m.rows - 1)];
            s[j] = __uint_as_float(v[j]) * factor * f.x * f.y;
          }
          if (!ok) return;
          if constexpr (kGated) {
            // a pair of lanes has gate and up of an output: the even one finishes the even rows, the odd one the odd rows
#pragma unroll
            for (int j = 0; j < S::kTurn; j += 2) {
              const float other = __shfl_xor_sync(0xffffffffu, lane & 1 ? s[j] : s[j + 1], 1);
              const int row = c + j + (lane & 1);
              const float out = lane & 1 ? mt_act<ACT>(other, s[j + 1], a) : mt_act<ACT>(s[j], other, a);
              if (row < m.rows && feature >> 1 < n_out) y[(size_t)(m.first + row) * ldy + (feature >> 1)] = from_f32<TO>(out);
            }
          } else {
#pragma unroll
            for (int j = 0; j < S::kTurn; ++j)
              if (c + j < m.rows && feature < n_out) y[(size_t)(m.first + c + j) * ldy + feature] = from_f32<TO>(mt_act<ACT>(s[j], 0.f, a));
          }
        });
      // Block r of a cluster finishes features r * per .. of the tile.
      const int log_splits = 31 - __clz(splits), per = 128 >> log_splits, stride = per + 4;
      if (splits > 1) {
        const int in = quarter * 32 + lane, owner = in >> (7 - log_splits);
        const uint32_t dst = map_to_cta(smem_u32(red + (size_t)rank * NT * stride + (in & (per - 1))), owner), bar = map_to_cta(red_bar, owner);
        const int sent = (m.rows + 7) & ~7;
        if (et == 0) mbar_expect_tx(red_bar, 128 * 4 * sent);      // (the stores themselves count on the owner's barrier: no fence, no arrivals)
        columns([&](int c, const uint32_t (&v)[S::kTurn]) {
#pragma unroll
          for (int j = 0; j < S::kTurn; ++j)
            if (j < 8 || c + j < sent) st_async_f32(dst + (c + j) * stride * 4, __uint_as_float(v[j]), bar);
        });
      }
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty_bar(b));
      if (++b == 2) { b = 0; acc_phase ^= 1; }
      if (splits > 1) {      // (a cluster has one tile: its sums' place is used once)
        if (!mbar_wait_cluster(red_bar, 0)) {
          if (a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00E5);
          ok = false;
        }
        const int outs = per >> kGated, o = et & (outs - 1), f = rank * per + (o << kGated), out = (m.feature + f) >> kGated;      // (f: in the tile)
        if (!ok || out >= n_out) continue;
        const float g_factor = a.w_factors[(size_t)m.expert * a.N + m.feature + f], u_factor = kGated ? a.w_factors[(size_t)m.expert * a.N + m.feature + f + 1] : 0.f;
#pragma unroll 4
        for (int c = et / outs; c < m.rows; c += 32 * S::kStorers / outs) {
          const float* from = red + (size_t)c * stride + (o << kGated);
          float g = from[0], u = from[kGated];
#pragma unroll
          for (int r = 1; r < 8; ++r)
            if (r < splits) {
              g += from[r * NT * stride];
              u += from[r * NT * stride + kGated];
            }
          const float2 f = factors[c];
          g = g * g_factor * f.x * f.y;
          u = u * u_factor * f.x * f.y;
          y[(size_t)(m.first + c) * ldy + out] = from_f32<TO>(mt_act<ACT>(g, u, a));
        }
      }
    }
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(a.tmem_cols) : "memory");
  }
}

template <int NT> static uint32_t mt_smem(int stages, int splits, int experts) {
  return 1024u + stages * MtShape<NT>::kStage + kMtBarBytes + 4 * (mt_red_floats<NT>(splits) + 4 * NT + 2 * (experts + 1));
}

// The blocks that share a tile's steps, where there is room for them beside the other tiles': 8, 4 or 2 if they are enough to pay for the exchange; of tiles of 128 rows, whose
// exchange is four times as long, at most 4, and none of few steps.  (us by 1 / 2 / 4 / 8 blocks a tile: 8 rows 512 -> 1,024 2.8 / 3.2 / 3.3 / 3.3, 1,024 -> 1,024 3.2 /
// 3.4 / 3.3 / 3.3, 2,048 -> 2,048 4.3 / 4.0 / 3.8 / 3.7, 4,096 -> 2,048 6.7 / 5.7 / 4.8 / 4.0, 4,096 -> 4,096 6.9 / 6.1 / 5.3 / 5.8, 4,096 -> 6,144 7.1 / 6.5 / 5.9 /
// 9.4, 14,336 -> 4,096 17.8 / 13.3 / 9.5 / 9.3; 64 rows 1,024 -> 1,302 6.2 / 5.2 / 4.5 / 5.8, 4,096 -> 4,096 9.0 / 7.5 / 7.0 / 17.5; 128 rows 4,096 -> 2,048
// 9.6 / 9.1 / 7.2 / 15.1; 333 rows 1,024 -> 1,302 6.8 / 7.6 / 7.4 / 20.9.)
static int mt_splits(int64_t tiles, int steps, int M, int blocks) {
  if (M > 32) return steps < (M <= 64 ? 4 : 8) ? 1 : tiles * 4 <= blocks ? 4 : tiles * 2 <= blocks ? 2 : 1;
  if (tiles * 8 <= (steps >= 32 ? blocks : blocks / 2) && steps >= 8) return 8;
  return steps < 4 ? 1 : tiles * 4 <= blocks ? 4 : tiles * 2 <= blocks ? 2 : 1;
}

// How a product runs: blocks in the grid, those that share a tile, steps of a block at most, stages of its ring; what a block takes of tensor memory and of shared memory.
struct MtPlan { int grid, splits, steps, stages; uint32_t tmem_cols, smem; };
template <int NT> static int mt_plan(int M, int N, int steps, int experts, MtPlan& p) {      // experts: 0 for one matrix
  using S = MtShape<NT>;
  constexpr int kBlocks = 148 * S::kPerSm;
  const int64_t row_tiles = experts ? M / NT + (M < experts ? M : experts) : ceil_div(M, NT), tiles = row_tiles * ceil_div(N, 128);
  p.splits = experts ? 1 : mt_splits(tiles, steps, M, kBlocks);
  if (tiles * p.splits > 0x7fffffff) return TIB_E_SIZE;
  p.grid = (int)(p.splits > 1 ? tiles * p.splits : tiles < kBlocks ? tiles : kBlocks);
  const int64_t most = (int64_t)ceil_div(steps, p.splits) * ceil_div64(tiles * p.splits, p.grid);
  p.steps = (int)(most < 0x7fffffff ? most : 0x7fffffff);
  p.stages = 1;
  while (p.stages < S::stages(p.splits) && p.stages < p.steps && mt_smem<NT>(p.stages + 1, p.splits, experts) <= (S::kPerSm > 1 ? 113u * 1024 : (uint32_t)kMostSmem)) ++p.stages;
  p.tmem_cols = p.splits > 1 ? 128 : 32;      // (in clusters: see smem_for_tmem)
  while (p.tmem_cols < S::scale_cols(p.splits) + 32 * p.stages) p.tmem_cols *= 2;
  p.smem = smem_for_tmem(mt_smem<NT>(p.stages, p.splits, experts), p.tmem_cols);
  return TIB_OK;
}
// Rows of a tile: 32 where all rows are one tile, else 128 (the tiles of their scales).  A tile's time is that of its weights: 8, 32, 33, 64 and 128 rows
// 4,096 -> 28,672 take 12.3, 13.9, 14.3, 15.8 and 16.9 us.
static int mt_tile_rows(int M) { return M <= 32 ? 32 : 128; }

template <int NT, int ACT, typename TO, bool MAKE>
static int launch_mt(MsArgs& a, void* y, int64_t ldy, cudaStream_t stream) {
  const int experts = a.offsets ? a.experts : 0;
  MtPlan plan;
  const int rc = mt_plan<NT>(a.M, a.N, a.steps, experts, plan);
  if (rc != TIB_OK) return rc;
  a.stages = plan.stages;
  a.tmem_cols = (int)plan.tmem_cols;
  auto kern = microscaled_tcgen05_kernel<NT, ACT, TO, MAKE>;
  static bool allowed[64];      // (by device: the attribute belongs to its context)
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && !(device < 64 && allowed[device])) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
  if (e != cudaSuccess) return (int)e;
  if (device < 64) allowed[device] = true;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(MtShape<NT>::kThreads);
  cfg.dynamicSmemBytes = plan.smem;
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
  e = cudaLaunchKernelEx(&cfg, kern, (const MsArgs)a, (TO*)y, ldy);
  if (e != cudaSuccess) return (int)e;
  TIB_LAUNCH_CHECK();
  return TIB_OK;
}

template <int NT, typename TO, bool MAKE>
static int launch_mt_act(int act, MsArgs& a, void* y, int64_t ldy, cudaStream_t stream) {
  switch (act) {
    case MOE_ACT_NONE: return launch_mt<NT, MOE_ACT_NONE, TO, MAKE>(a, y, ldy, stream);
    case MOE_ACT_RELU2: return launch_mt<NT, MOE_ACT_RELU2, TO, MAKE>(a, y, ldy, stream);
    case MOE_ACT_SILU: return launch_mt<NT, MOE_ACT_SILU, TO, MAKE>(a, y, ldy, stream);
    case MOE_ACT_GELU: return launch_mt<NT, MOE_ACT_GELU, TO, MAKE>(a, y, ldy, stream);
    case MOE_ACT_GLU_CLAMP: return launch_mt<NT, MOE_ACT_GLU_CLAMP, TO, MAKE>(a, y, ldy, stream);
    default: return launch_mt<NT, MOE_ACT_SWIGLU, TO, MAKE>(a, y, ldy, stream);
  }
}

}  // namespace tib

using namespace tib;

// Where a block's threads find the rows' largest numbers with one round of loads, and have a tile each.  (One kernel / two, us on the device: 1 row 1,024 -> 1,024 3.5 / 4.4, 8 rows
// 3.8 / 4.7; 4 rows 2,048 -> 2,048 4.3 / 4.9; 2 rows 4,096 -> 4,096 6.5 / 6.5; 1 row 4,096 -> 28,672 14.6 / 14.5, 2 rows 15.2 / 14.8; 1 row 8,192 -> 8,192 10.4 / 10.2; where calls
// are bound by the host 8.5 / 12.1 each.  With more rounds every block's reading of all rows shows: 4 rows 4,096 -> 4,096 8.0 / 6.6, 1 row 14,336 -> 4,096 11.2 / 10.5.)
bool tib::ms_makes_rows(int M, int N, int K) {
  MtPlan p{};
  return M <= 8 && K % 8 == 0 && K <= 1024 << mt_more_loads(M) && mt_plan<32>(M, N, ms_steps(K), 0, p) == TIB_OK && p.grid == ceil_div(N, 128) * p.splits;
}

int tib::ms_product_tcgen05(MsArgs& a, int act, void* y, int y_dtype, int64_t ldy, cudaStream_t stream) {
  if (a.experts > kMtMaxExperts || (int64_t)a.experts * ceil_div(a.N, 128) * a.steps > 0x7fffffff) return TIB_E_SIZE;
#define TIB_MT_GO(NT, MAKE) \
  return y_dtype == TIB_BF16 ? launch_mt_act<NT, __nv_bfloat16, MAKE>(act, a, y, ldy, stream) : launch_mt_act<NT, float, MAKE>(act, a, y, ldy, stream)
  if (a.made) TIB_MT_GO(32, true);
  if (mt_tile_rows(a.M) == 32) TIB_MT_GO(32, false);
  TIB_MT_GO(128, false);
#undef TIB_MT_GO
}

static int mt_plan_of(int M, int N, int steps, int experts, MtPlan& p) {
  return mt_tile_rows(M) == 32 ? mt_plan<32>(M, N, steps, experts, p) : mt_plan<128>(M, N, steps, experts, p);
}
int tib::ms_plan_tcgen05(int M, int N, int steps, int experts, int* plan) {
  MtPlan p{};
  const int rc = mt_plan_of(M, N, steps, experts, p);
  plan[0] = mt_tile_rows(M); plan[1] = p.splits; plan[2] = p.steps; plan[3] = p.stages;
  return rc;
}
int tib::ms_room_tcgen05(int M, int N, int steps, int experts, int* room) {
  MtPlan p{};
  const int rc = mt_plan_of(M, N, steps, experts, p);
  room[0] = (int)p.tmem_cols; room[1] = (int)p.smem;
  return rc;
}
