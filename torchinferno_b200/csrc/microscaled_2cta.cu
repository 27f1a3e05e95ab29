// Products of 4-bit microscaled operands for many rows, plain or sorted by expert, on pairs of SMs: out[M, N] = x . w^T with
// `tcgen05.mma.cta_group::2`, where
//     out[m, n] = act(r[m] f[n] (sum over runs b of s[m, b] S[n, b] (sum over the 16 columns of run b of x[m, k] w[n, k]))).
//
// Two blocks (a cluster of two) compute a tile of 256 rows x 256 features: block r holds rows r * 128 .. of the x slice and features r * 128 .. of the w
// slice, and gets rows r * 128 .. of the accumulator, which needs the scales of its own rows and of all 256 features.  A step is 256 columns: the 128-byte
// row of the swizzle, twelve copies of scales to tensor memory, four MMAs.  The accumulator (256 columns) stays in tensor memory for the whole sum; beside it
// every stage of the ring has 48 columns for its scales.
//   warp 0       TMA producer into a ring of five stages, the first weights ahead of the end of the kernel before      warp 1 (of the even block)   copies scales and issues the MMAs; either owns its block's TMEM
//   warps 4..11  epilogue, 32 rows x 128 features each: read into registers at once, so that the next tile's MMAs may begin, then finished.  These take registers
//                that the first four warps give up (168 a thread at launch, 40 + 2 x 232 after)
// What bounds it: the step, and behind the last of a tile its reading.  8,192 rows -> 28,672: 146, 368 and 663 us at 1,024, 4,096 and 8,192 columns, so 0.37 us a step of
// 256 (some 690 cycles, where the MMAs take 512) and 1.6 us a tile beside them.  Without the copies from memory a step takes 0.31 us (the MMAs read 32 KB of shared memory a step,
// the scales' copies 6, and 38 KB are written: 76 KB for a port of 128 bytes a cycle are 594), and without the outputs a tile costs 0.3 us: those are 64 KB a block through
// the same paths.  The gated product of 8,192 rows 4,096 -> 2 x 14,336 takes 0.34 ms, 5,600 TFLOP/s, 0.36 with its rows' codes, in a row under the power limit 0.42.  (What
// took it there from 0.62 ms: see ms_umma; the features' factors read from shared memory in place of global, 0.38 to 0.37; a tile's factors asked for a tile ahead, at 1,024
// columns 154 to 146.)
// Every wait is bounded and reports in error_word; no block leaves before its partner is done and what was sent to it has come; every copy lands in the block that
// issued it.
#include "microscaled.cuh"

namespace tib {

constexpr int kM2Stages = 5, kM2Threads = 384;
constexpr uint32_t kM2Half = kMsTileRows * kMsStepBytes, kM2Stage = 2 * kM2Half + 3 * kMsStepScales;      // x, w, scales of x, of w's two tiles
constexpr uint32_t kM2Smem = kM2Stages * kM2Stage + 1024 /* alignment */ + 256 /* barriers */ + 8 * 4096 /* outputs */ + 2 * 1024 /* factors */;
constexpr int kM2MaxExperts = (kMostSmem - (int)kM2Smem) / 8 - 1;      // (two numbers each in what is left of shared memory)
constexpr uint32_t kM2Idesc = kMsIdesc | ((256u >> 3) << 17) | ((256u >> 4) << 24);      // N = 256, M = 256 over the pair
constexpr uint32_t kM2ScaleCols = 256;      // where the stages' scales begin in tensor memory: 16 columns of x's, 32 of w's each
static_assert(kM2ScaleCols + 48 * kM2Stages <= 512, "tensor memory");

struct M2Tile { int expert, first, rows, group, scale_tile, n_tile; };      // rows first .. first + rows - 1 of x (at most 256), features n_tile * 256 ..

// Persistent: pair p walks the tiles t = p, p + pairs, ...  Of one matrix, tile t is row tile t % m_tiles of feature tile t / m_tiles, so pairs that run
// together share slices of w; of rows sorted by expert, feature tiles run fastest.
template <int ACT, typename TO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kM2Threads, 1)
microscaled_2cta_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_xs,
                        const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ MsArgs a, TO* __restrict__ out, int64_t ldo, int wide_stores) {
  constexpr bool kGated = moe_act_gated(ACT);
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = base + kM2Stages * kM2Stage;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kM2Stages + s); };
  const uint32_t acc_full_bar = bars + 8u * (2 * kM2Stages), acc_empty_bar = acc_full_bar + 8, tmem_slot = acc_full_bar + 16;
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - smem_u32(smem_raw)));

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();                    // 0: the even block of the pair, which issues the MMAs
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int n_tiles = (a.N + 255) >> 8;
  float* tile_factors = reinterpret_cast<float*>(smem_raw + (bars - smem_u32(smem_raw)) + 256 + 8 * 4096);  // [2][256] the features', of two tiles in turn
  int* tiles_before = reinterpret_cast<int*>(tile_factors + 512);                                           // [experts + 1] where rows are sorted, and
  int* first_row = tiles_before + a.experts + 1;                                                            // [experts + 1] their offsets

  if (threadIdx.x == 0) {
    for (int s = 0; s < kM2Stages; ++s) {
      mbar_init(full_bar(s), 1);          // (used in the even block: its producer's arrival, plus the bytes of both)
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(acc_full_bar, 1);
    mbar_init(acc_empty_bar, 16);         // (used in the even block: eight epilogue warps of each block)
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tmem_slot), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  if (a.offsets) pdl_wait();                               // (of one matrix, each warp waits where it first needs what the kernel ahead leaves)
  if (a.offsets && warp == 0) {                            // the experts' row tiles, summed
    int before = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane, begin = e < a.experts ? bs_offset(a.offsets, e, a.M) : 0;
      int sum = e < a.experts ? (max(0, bs_offset(a.offsets, e + 1, a.M) - begin) + 255) >> 8 : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      if (e < a.experts) tiles_before[e + 1] = before + sum, first_row[e] = begin;
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) tiles_before[0] = 0, first_row[a.experts] = bs_offset(a.offsets, a.experts, a.M);
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  cluster_sync_all();                                      // both blocks have their barriers before either is signalled
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  pdl_trigger();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot_ptr, 0);
  const int m_tiles = a.offsets ? tiles_before[a.experts] : (a.M + 255) >> 8, num_tiles = m_tiles * n_tiles;
  auto tile_of = [&](int t) {
    M2Tile m;
    if (!a.offsets) {
      m.n_tile = t / m_tiles;
      m.expert = 0;
      m.first = (t - m.n_tile * m_tiles) * 256;
      m.rows = min(256, a.M - m.first);
      m.scale_tile = m.first >> 7;
      m.group = m.first >> 3;
      return m;
    }
    const int row_tile = t / n_tiles;
    m.n_tile = t - row_tile * n_tiles;
    int lo = 0, hi = a.experts;                            // tiles_before[lo] <= row_tile < tiles_before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tiles_before[mid] <= row_tile) lo = mid; else hi = mid;
    }
    const int j = row_tile - tiles_before[lo];
    m.expert = lo;
    m.first = first_row[lo] + j * 256;
    m.rows = min(256, first_row[lo + 1] - m.first);
    m.scale_tile = ms_first_tile(first_row[lo], lo) + 2 * j;
    m.group = ms_first_group(first_row[lo], lo) + 32 * j;
    return m;
  };

  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;\n");
    const int quarter = warp & 3, half = (warp - 4) >> 2, et = threadIdx.x - 128;
    uint32_t acc_phase = 0;
    bool ok = true;
    // A tile's factors (of a feature, of this thread's row and of its pair) are asked for while the tile before is finished.
    float w_factor = 0.f, x_factor = 0.f, pair_factor = 1.f;
    auto ask = [&](const M2Tile& m) {
      const int row = min(m.first + (int)rank * 128 + quarter * 32 + lane, m.first + m.rows - 1);
      w_factor = a.w_factors[(size_t)m.expert * a.N + min(m.n_tile * 256 + et, a.N - 1)];
      x_factor = a.x.factors[row];
      if (a.row_scale) pair_factor = a.row_scale[bs_pair(a.order, row, a.M)];
    };
    M2Tile next = {};
    if (!a.offsets) pdl_wait();
    if (pair < num_tiles) ask(next = tile_of(pair));
    for (int t = pair; t < num_tiles; t += pairs, acc_phase ^= 1) {
      const M2Tile m = next;
      const int in_tile = (int)rank * 128 + quarter * 32 + lane, row = m.first + in_tile, last = m.first + m.rows;      // (rows from `last` on are not stored)
      const int col0 = m.n_tile * 256 + half * 128;
      tile_factors[acc_phase * 256 + et] = w_factor;
      const float2 of_row = a.row_scale ? ms_row_factors(x_factor, pair_factor) : ms_row_factors(x_factor);
      const f32x2 ahead2 = f2_pack(of_row.x, of_row.x), behind2 = f2_pack(of_row.y, of_row.y);
      if (t + pairs < num_tiles) ask(next = tile_of(t + pairs));
      asm volatile("bar.sync 1, 256;\n" ::: "memory");      // (the last tile but one is finished: its factors have been read)
      if (ok && !mbar_wait_warp(acc_full_bar, acc_phase)) {
        if (a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00F3);
        ok = false;
      }
      if (!ok) continue;
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      uint32_t v[4][32];
      const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld32(acc + 32 * i, v[i]);
      asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      __syncwarp();
      // (what this orders is the reading of tensor memory, which tcgen05.fence has ordered: no fence of the cluster)
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(map_to_cta(acc_empty_bar, 0)) : "memory");
      f32x2 sum[64];
      const ulonglong2* factors2 = reinterpret_cast<const ulonglong2*>(tile_factors + acc_phase * 256 + half * 128);
#pragma unroll
      for (int c = 0; c < 64; c += 2) {      // (by the row: see ms_row_factors)
        const ulonglong2 f = factors2[c >> 1];
        sum[c] = f2_mul(f2_mul(f2_pack(__uint_as_float(v[c >> 4][2 * c & 31]), __uint_as_float(v[c >> 4][(2 * c & 31) + 1])), ahead2), f.x);
        sum[c + 1] = f2_mul(f2_mul(f2_pack(__uint_as_float(v[c >> 4][(2 * c & 31) + 2]), __uint_as_float(v[c >> 4][(2 * c & 31) + 3])), ahead2), f.y);
      }
      if (__any_sync(0xffffffffu, of_row.y != 1.f)) {      // (a pair's factor, or a row at the ends of the range)
#pragma unroll
        for (int c = 0; c < 64; ++c) sum[c] = f2_mul(sum[c], behind2);
      }
      // A row's outputs lie in one thread: a warp's 32 rows cross its 4 KB of shared memory, 128 bytes of each at a time (16-byte pieces, swizzled by row),
      // and leave as whole lines.
      constexpr int kOut = kGated ? 64 : 128, kVec = 16 / sizeof(TO), kTurn = 8 * kVec;      // outputs of a thread, a piece, a turn
      const int first = col0 >> kGated, n_out = a.N >> kGated;
      unsigned char* mine = smem_raw + (base - smem_u32(smem_raw)) + kM2Stages * kM2Stage + 256 + (warp - 4) * 4096;
#pragma unroll
      for (int turn = 0; turn < kOut / kTurn; ++turn) {
        if (first + turn * kTurn >= n_out) break;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          float y[kVec];
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const int c = turn * kTurn + p * kVec + j;
            float lo, hi;
            f2_unpack(sum[kGated ? c : c >> 1], lo, hi);
            y[j] = kGated ? bs_gated<ACT>(lo, hi, a.limit, a.alpha) : bs_act<ACT>(c & 1 ? hi : lo);
          }
          uint4 w;
          if constexpr (sizeof(TO) == 2) {
            __nv_bfloat162 b2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b2[j] = __floats2bfloat162_rn(y[2 * j], y[2 * j + 1]);
            w = *reinterpret_cast<const uint4*>(b2);
          } else {
            w = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
          }
          *reinterpret_cast<uint4*>(mine + lane * 128 + ((p ^ (lane & 7)) << 4)) = w;
        }
        __syncwarp();
        if (wide_stores) {
          const int p = lane & 7, col = first + turn * kTurn + p * kVec;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3);
            const uint4 w = *reinterpret_cast<const uint4*>(mine + r * 128 + ((p ^ (r & 7)) << 4));
            if (row - lane + r >= last) continue;
            TO* dst = out + (size_t)(row - lane + r) * ldo + col;
            if (col + kVec <= n_out) *reinterpret_cast<uint4*>(dst) = w;
            else {
              const TO* one = reinterpret_cast<const TO*>(&w);
#pragma unroll
              for (int j = 0; j < kVec; ++j)
                if (col + j < n_out) dst[j] = one[j];
            }
          }
        } else {      // (rows that are not 16-byte aligned: consecutive lanes write consecutive outputs of one row)
#pragma unroll 1
          for (int r = 0; r < min(32, last - (row - lane)); ++r) {
#pragma unroll
            for (int c = lane; c < kTurn; c += 32) {
              const TO o = *reinterpret_cast<const TO*>(mine + r * 128 + (((c / kVec) ^ (r & 7)) << 4) + (c % kVec) * sizeof(TO));
              const int col = first + turn * kTurn + c;
              if (col < n_out) out[(size_t)(row - lane + r) * ldo + col] = o;
            }
          }
        }
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n");
    if (warp == 0) {
      const uint32_t leader = umma_leader();
      int ahead = 0, it = 0, s = 0;
      uint32_t phase = 1;
      bool ok = true;
      const int blocks = (a.N + 127) >> 7;
      // (a pair's second tile of features may lie behind the matrix: it reads the last one instead, which is not stored)
      auto w_at = [&](const M2Tile& m, int half) { return (m.expert * blocks + min(m.n_tile * 2 + half, blocks - 1)) * a.steps; };
      // (a step's five copies; x's last two by themselves where the weights' are on their way already)
      auto ask = [&](int w0, int s0, int s1, int xs0, int group, int step, int s, bool w, bool x) {
        if (w && rank == 0) mbar_expect_tx(full_bar(s), 2 * kM2Stage);
        const uint32_t bar0 = map_to_cta(full_bar(s), 0), stage = base + s * kM2Stage, scales = stage + 2 * kM2Half;
        if (x) pair_tma_load(stage, &map_x, 0, step * a.x.groups + group, bar0);
        if (w) pair_tma_load(stage + kM2Half, &map_w, 0, (w0 + step) << 4, bar0);
        if (x) pair_tma_load(scales, &map_xs, 0, (xs0 + step) << 2, bar0);
        if (w) {
          pair_tma_load(scales + kMsStepScales, &map_ws, 0, (s0 + step) << 2, bar0);
          pair_tma_load(scales + 2 * kMsStepScales, &map_ws, 0, (s1 + step) << 2, bar0);
        }
      };
      if (!a.offsets) {      // the first weights: they do not wait for the kernel ahead
        for (int t = pair; t < num_tiles && ahead < kM2Stages; t += pairs) {
          const M2Tile m = tile_of(t);
          for (int step = 0; step < a.steps && ahead < kM2Stages; ++step, ++ahead)
            if (leader) ask(w_at(m, (int)rank), w_at(m, 0), w_at(m, 1), 0, 0, step, ahead, true, false);
        }
        pdl_wait();
      }
      for (int t = pair; t < num_tiles && ok; t += pairs) {
        const M2Tile m = tile_of(t);
        const int w0 = w_at(m, (int)rank), s0 = w_at(m, 0), s1 = w_at(m, 1), xs0 = (m.scale_tile + (int)rank) * a.steps;
        const int group = m.group + (int)rank * 16;        // (behind the tile's rows come others', which are not stored, or zeros)
        for (int step = 0; step < a.steps; ++step, ++it) {
          if (it < ahead) {
            if (leader) ask(w0, s0, s1, xs0, group, step, s, false, true);
          } else {
            if (!mbar_wait_warp(empty_bar(s), phase)) {
              if (a.error_word && leader) atomicExch(a.error_word, 0x7C00F1);
              ok = false;
              break;
            }
            if (leader) ask(w0, s0, s1, xs0, group, step, s, true, true);
          }
          __syncwarp();
          if (++s == kM2Stages) { s = 0; phase ^= 1; }
        }
      }
      // The even block's last releases of the stages arrive here as well: they have come before this block leaves.
      for (int i = 0; i < kM2Stages && ok; ++i) {
        if (!mbar_wait_warp(empty_bar(s), phase)) {
          if (a.error_word && leader) atomicExch(a.error_word, 0x7C00F1);
          ok = false;
        }
        if (++s == kM2Stages) { s = 0; phase ^= 1; }
      }
    } else if (warp == 1 && rank == 0) {
      const uint32_t leader = umma_leader();
      if (!a.offsets) pdl_wait();      // (the bounded waits begin when the kernel ahead is over)
      int s = 0;
      uint32_t phase = 0, acc_phase = 1;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += pairs) {
        if (!__all_sync(0xffffffffu, pair_wait(acc_empty_bar, acc_phase))) {      // both blocks have read the accumulator
          if (a.error_word && leader) atomicExch(a.error_word, 0x7C00F4);
          break;
        }
        acc_phase ^= 1;
        for (int step = 0; step < a.steps; ++step) {
          if (!__all_sync(0xffffffffu, pair_wait(full_bar(s), phase))) {
            if (a.error_word && leader) atomicExch(a.error_word, 0x7C00F2);
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          const uint32_t stage = base + s * kM2Stage, scales = stage + 2 * kM2Half, columns = tmem_base + kM2ScaleCols + 48 * s;
          const uint32_t x_src = umma_low_k128(stage), w_src = x_src + (kM2Half >> 4);
          if (leader) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              ms_copy_scales<2>(columns + 4 * k, scales + kMsChunkBytes * k);
              ms_copy_scales<2>(columns + 16 + 8 * k, scales + kMsStepScales + kMsChunkBytes * k);
              ms_copy_scales<2>(columns + 20 + 8 * k, scales + 2 * kMsStepScales + kMsChunkBytes * k);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) ms_umma<2>(tmem_base, x_src + 2 * k, w_src + 2 * k, kM2Idesc, columns + 4 * k, columns + 16 + 8 * k, step != 0 || k != 0);
            pair_commit_both(empty_bar(s));      // the stage is free in both blocks once these MMAs have read it
          }
          __syncwarp();
          if (++s == kM2Stages) { s = 0; phase ^= 1; }
        }
        if (leader) pair_commit_both(acc_full_bar);
        __syncwarp();
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  cluster_sync_all();   // neither block leaves (or frees tensor memory) while its partner may still signal it
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// Pieces of so many bytes (at most 1024) side by side in memory, read so many at a time.
static int m2_map(CUtensorMap* map, const void* ptr, int64_t pieces, int bytes, int at_a_time) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return TIB_E_ARG;
  const cuuint64_t dims[2] = {(cuuint64_t)bytes / 4, (cuuint64_t)pieces};
  const cuuint64_t strides[1] = {(cuuint64_t)bytes};
  const cuuint32_t box[2] = {(cuuint32_t)bytes / 4, (cuuint32_t)at_a_time};
  const cuuint32_t elem[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TIB_OK : TIB_E_ARG;
}

static_assert(kM2Smem >= tmem_share_smem(512), "see smem_for_tmem");
static uint32_t m2_smem(int experts) { return kM2Smem + (experts ? 8 * (experts + 1) : 0); }

static int64_t m2_tiles(int M, int N, int experts) {      // at most; experts: 0 for one matrix
  return (int64_t)(experts ? M / 256 + (M < experts ? M : experts) : ceil_div(M, 256)) * ceil_div(N, 256);
}

template <int ACT, typename TO>
static int launch_m2(const CUtensorMap (&maps)[4], const MsArgs& a, void* out, int64_t ldo, cudaStream_t stream) {
  auto kern = microscaled_2cta_kernel<ACT, TO>;
  static bool allowed[64];      // (by device: the attribute belongs to its context)
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && !(device < 64 && allowed[device])) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
  if (e != cudaSuccess) return (int)e;
  if (device < 64) allowed[device] = true;
  const int64_t tiles = m2_tiles(a.M, a.N, a.offsets ? a.experts : 0);
  if (tiles > 0x7fffffff) return TIB_E_SIZE;
  const int wide = ((uintptr_t)out & 15) == 0 && (ldo * sizeof(TO)) % 16 == 0;
  TIB_LAUNCH_DEPENDENT(kern, 2 * (int)(tiles < 74 ? tiles : 74), kM2Threads, m2_smem(a.offsets ? a.experts : 0), stream, maps[0], maps[1], maps[2], maps[3], a,
                       (TO*)out, ldo, wide);
  return TIB_OK;
}

}  // namespace tib

using namespace tib;

// Whether a product runs here (experts: 0 for one matrix).  Of one matrix: more than one tile of 128 rows, and enough tiles of 128 x 128 to keep pairs of SMs busy, the more
// the longer they are.  (us, tiles of 128 / pairs: 4,096 -> 28,672 128 rows 16.9 / 19.5, 192 rows 25.8 / 20.0; 300 rows 2,048 -> 4,096 7.9 / 8.0; 1,024 rows
// 1,024 -> 1,024 10.1 / 7.2; 4,096 -> 4,096 256 rows 10.6 / 10.3, 512 rows 10.8 / 10.4, 768 rows 15.3 / 11.0; 200 rows 2,048 -> 1,302 6.8 / 10.1; 512 rows 8,192 ->
// 4,096 15.0 / 15.1; 14,336 -> 4,096 256 rows 16.7 / 22.3, 512 rows 21.5 / 22.7.)  Of rows by expert: from 16 an expert on, on average.  (32 experts 2,048 -> 1,024 with
// their rows' codes, 4 choices a token: 64 tokens 14.3 / 17.0, 128 18.0 / 17.7, 256 19.4 / 18.4, 1,024 28.6 / 24.3, 2,048 44.4 / 34.0; gated 64 22.8 / 22.2, 128 27.1 / 24.3, 512
// 39.5 / 28.3; 8 experts 1,024 -> 1,024 16 rows an expert 9.6 / 10.3.)
constexpr int kM2ExpertRows = 16;
bool tib::ms_on_pairs_of_sms(int M, int N, int steps, int experts) {
  if (experts) return M >= (int64_t)experts * kM2ExpertRows && experts <= kM2MaxExperts;
  return M > 128 && (int64_t)ceil_div(M, 128) * ceil_div(N, 128) >= (steps <= 16 ? 64 : steps <= 32 ? 128 : 149);
}

int tib::ms_product_2cta(const MsArgs& a, int act, void* out, int out_dtype, int64_t ldo, cudaStream_t stream) {
  if (a.offsets && a.experts > kM2MaxExperts) return TIB_E_SIZE;
  const int64_t w_steps = (int64_t)a.experts * ceil_div(a.N, 128) * a.steps, x_tiles = ceil_div(a.M, 128) + (a.offsets ? a.experts : 0);
  if (w_steps > (0x7fffffff >> 4) || (int64_t)a.x.groups * a.steps > 0x7fffffff || x_tiles * a.steps > (0x7fffffff >> 2)) return TIB_E_SIZE;
  CUtensorMap maps[4];
  int rc = m2_map(&maps[0], a.x.codes, (int64_t)a.x.groups * a.steps, kMsGroupBytes, 16);
  if (rc == TIB_OK) rc = m2_map(&maps[1], a.w, w_steps * 16, kMsGroupBytes, 16);
  if (rc == TIB_OK) rc = m2_map(&maps[2], a.x.scales, x_tiles * a.steps * 4, kMsChunkBytes, 4);
  if (rc == TIB_OK) rc = m2_map(&maps[3], a.w_scales, w_steps * 4, kMsChunkBytes, 4);
  if (rc != TIB_OK) return rc;
#define TIB_M2_GO(ACT) \
  case ACT: return out_dtype == TIB_BF16 ? launch_m2<ACT, __nv_bfloat16>(maps, a, out, ldo, stream) : launch_m2<ACT, float>(maps, a, out, ldo, stream)
  switch (act) {
    TIB_M2_GO(MOE_ACT_NONE);
    TIB_M2_GO(MOE_ACT_RELU2);
    TIB_M2_GO(MOE_ACT_SILU);
    TIB_M2_GO(MOE_ACT_GELU);
    TIB_M2_GO(MOE_ACT_GLU_CLAMP);
    TIB_M2_GO(MOE_ACT_SWIGLU);
  }
#undef TIB_M2_GO
  return TIB_E_SIZE;
}

int tib::ms_plan_2cta(int M, int N, int steps, int experts, int* plan) {
  const int64_t tiles = m2_tiles(M, N, experts), most = steps * ceil_div64(tiles, tiles < 74 ? tiles : 74);
  plan[0] = 256; plan[1] = 1; plan[2] = (int)(most < 0x7fffffff ? most : 0x7fffffff); plan[3] = kM2Stages;
  return TIB_OK;
}

int tib::ms_room_2cta(int experts, int* room) {
  room[0] = 512; room[1] = (int)m2_smem(experts);
  return TIB_OK;
}
