// Products of 8-bit block-scaled operands for many rows, plain or sorted by expert, on pairs of SMs: out[M, N] = x . w^T with
// `tcgen05.mma.cta_group::2`, where
//     out[m, n] = sum over runs b of s[m, b] S[n's block, b] (sum over the 128 columns of run b of x[m, k] w[n, k]).
//
// Two blocks (a cluster of two) compute a tile of 256 rows x 256 features, as in gemm_tcgen05_2cta.cu: block r holds rows r * 128 .. of the
// x slice and features r * 128 .. of the w slice, and gets rows r * 128 .. of the accumulator.  A step is one run: 128 columns, the 128-byte row of the
// swizzle, four MMAs into one of two accumulators of 256 columns.  The sums over runs are taken in registers, since every run has its own scales:
// eight warps, 32 rows x 128 features each, read the accumulator in pieces of 16 columns, the next piece on its way under the multiply-adds of
// the last, and add it to 128 sums a thread, times the scale of (its row, run) and (the features' block, run).  Two sums are one packed
// multiply-add; in a matrix of (gate, up) row pairs the two have different scales, which the packed form takes as it comes.
//   warp 0       TMA producer into a ring of six stages      warp 1 (of the even block)   issues the MMAs; either owns its block's TMEM
//   warps 4..11  sums, then the epilogue with its activation.  These take registers that the first four warps give up (168 a thread at launch,
//                40 + 2 x 232 after)
// What bounds it: the step.  It takes 880 to 930 cycles of the warp that issues the MMAs, whose own time is 537: 135 to 160 in the wait for operands,
// 190 to 250 in that for an accumulator to be read, the rest in issuing.  Without the sums it takes 700, the sums alone 340.  (The bf16 kernel of the same tiles,
// whose accumulator changes hands once a tile and not once a step, takes about 550.)  8,192 rows 4,096 -> 2 x 14,336 with silu(gate) * up: 0.90 ms,
// 2,140 TFLOP/s (1.03 to 1.07 ms, 1,800 to 1,870 under the power limit); 2,048 rows 4,096 -> 6,144 with its codes 58 to 60 us, 1,740, a third round of tiles included that
// is 0.6 full.  Tried: pieces of 32 columns (the scales' registers spilled, and every step waited for their loads: 1.10 ms), waits by polling without a time hint (no gain).
// Every wait is bounded and reports in error_word; no block leaves before its partner is done and what was sent to it has come; every copy lands in the block that
// issued it.
#include "block_scaled.cuh"
#include "cluster.cuh"

namespace tib {

constexpr int kB2Stages = 6, kB2Threads = 384;
constexpr uint32_t kB2Half = 128 * kBlk, kB2Stage = 2 * kB2Half;
constexpr uint32_t kB2Smem = kB2Stages * kB2Stage + 1024 /* alignment */ + 256 /* barriers */ + 8 * 4096 /* outputs */;
constexpr int kB2MaxExperts = (kMostSmem - (int)kB2Smem) / 8 - 1;      // (two numbers each in what is left of shared memory)
// D fp32, A and B e4m3, both K-major, N = 256, M = 256 over the pair
constexpr uint32_t kB2Idesc = (1u << 4) | ((256u >> 3) << 17) | ((256u >> 4) << 24);

__device__ __forceinline__ void b2_umma(uint32_t leader, uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p, q;\n.reg .b64 a, b;\nmov.b64 a, {%1, %6};\nmov.b64 b, {%2, %6};\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
               "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, p;\n}\n"
               ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(kB2Idesc), "r"(accumulate), "r"(leader), "r"(kUmmaDescHigh) : "memory");
}
// An arrival at the even block's barrier without a fence of the cluster: what it orders is the reading of tensor memory, which tcgen05.fence has ordered.
// (With .release.cluster every step waited for the warp's whole memory traffic, the largest of the kernel's stalls.)
__device__ __forceinline__ void b2_arrive_even(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_bar) : "memory");
}

struct B2Args {
  const unsigned char* x;      // codes [M, runs * 128]
  const unsigned char* w;      // codes in blocks
  BsFar far;
  const float* x_scales;       // [runs, lds]
  int64_t lds;
  const float* w_scales;       // [rows of scales, runs]
  int scale_rows, pairs, M, N, runs;
  const int* offsets;          // [experts + 1] of rows sorted by expert, or null: one matrix
  const int* order;
  int experts;
  MoeEpilogue ep;
  int* error_word;
};

static_assert(2 * sizeof(CUtensorMap) + sizeof(B2Args) + 20 <= 416, "the kernel's parameters (see block_scaled_tcgen05.cu)");

struct B2Tile { int expert, first, rows, n_tile; };      // rows first .. first + rows - 1 of x (at most 256), features n_tile * 256 ..

// Rows row0 .. of a warp in a tile whose outputs are `first` ..: those outputs that have a far scale, made again, a lane an output.
template <int ACT, typename TO>
__device__ __noinline__ void b2_rows_apart(const B2Args* args, int row0, int rows, int expert, int first, TO* __restrict__ out, int64_t ldo) {
  const B2Args& a = *args;
  constexpr int kGated = moe_act_gated(ACT);
  const int lane = threadIdx.x & 31;
  bool outside = false;
  if (lane < rows)
    for (int b = 0; b < a.runs; ++b) outside |= a.far.outside(a.x_scales[(size_t)b * a.lds + row0 + lane]);
  for (uint32_t rest = __ballot_sync(0xffffffffu, outside); rest; rest &= rest - 1) {
    const int r = row0 + __ffs(rest) - 1;
    BsApart<uint8_t> apart;
    apart.x = a.x + (size_t)r * a.runs * kBlk;
    apart.x_scales = a.x_scales + r;
    apart.lds = a.lds; apart.pairs = a.pairs; apart.runs = a.runs; apart.K = 0; apart.act = ACT;
    apart.limit = a.ep.limit; apart.alpha = a.ep.alpha;
    apart.row_scale = a.ep.row_scale ? a.ep.row_scale[bs_pair(a.order, r, a.M)] : 1.f;
    apart.w = a.w + ((size_t)expert * ((a.N + 127) >> 7) * a.runs << 14);
    apart.w_scales = a.w_scales + (size_t)expert * a.scale_rows * a.runs;
    for (int c = first + lane; c < min(first + (128 >> kGated), a.N >> kGated); c += 32) bs_output_apart<uint8_t, TO>(apart, c, out + (size_t)r * ldo);
  }
}

// Persistent: pair p walks the tiles t = p, p + pairs, ...  Of one matrix, tile t is row tile t % m_tiles of feature tile t / m_tiles, so pairs that run
// together share slices of w; of rows sorted by expert, feature tiles run fastest.
template <int ACT, typename TO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kB2Threads, 1)
block_scaled_2cta_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ B2Args a,
                         TO* __restrict__ out, int64_t ldo, int wide_stores) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = base + kB2Stages * kB2Stage;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kB2Stages + s); };
  auto acc_full_bar = [&](int b) { return bars + 8u * (2 * kB2Stages + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * kB2Stages + 2 + b); };
  const uint32_t tmem_slot = bars + 8u * (2 * kB2Stages + 4);
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - smem_u32(smem_raw)));

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();                    // 0: the even block of the pair, which issues the MMAs
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int n_tiles = (a.N + 255) >> 8;
  int* tiles_before = reinterpret_cast<int*>(smem_raw + (bars - smem_u32(smem_raw)) + 256 + 8 * 4096);      // [experts + 1] where rows are sorted, and
  int* first_row = tiles_before + a.experts + 1;                                                            // [experts + 1] their offsets

  if (threadIdx.x == 0) {
    for (int s = 0; s < kB2Stages; ++s) {
      mbar_init(full_bar(s), 1);          // (used in the even block: its producer's arrival, plus the bytes of both)
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);
      mbar_init(acc_empty_bar(b), 16);    // (used in the even block: eight summing warps of each block)
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tmem_slot), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
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
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot_ptr, 0);
  const int m_tiles = a.offsets ? tiles_before[a.experts] : (a.M + 255) >> 8, num_tiles = m_tiles * n_tiles;
  auto tile_of = [&](int t) {
    B2Tile m;
    if (!a.offsets) {
      m.n_tile = t / m_tiles;
      m.expert = 0;
      m.first = (t - m.n_tile * m_tiles) * 256;
      m.rows = min(256, a.M - m.first);
      return m;
    }
    const int row_tile = t / n_tiles;
    m.n_tile = t - row_tile * n_tiles;
    int lo = 0, hi = a.experts;                            // tiles_before[lo] <= row_tile < tiles_before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tiles_before[mid] <= row_tile) lo = mid; else hi = mid;
    }
    m.expert = lo;
    m.first = first_row[lo] + (row_tile - tiles_before[lo]) * 256;
    m.rows = min(256, first_row[lo + 1] - m.first);
    return m;
  };

  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;\n");
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    int b = 0;
    uint32_t acc_phase = 0;
    bool ok = true, outside = false;           // (outside: a run of one of this thread's rows, of BsFar's range)
    for (int t = pair; t < num_tiles && ok; t += pairs) {
      const B2Tile m = tile_of(t);
      const int in_tile = (int)rank * 128 + quarter * 32 + lane, row = m.first + in_tile, last = m.first + m.rows;      // (rows from `last` on are not stored)
      const int col0 = m.n_tile * 256 + half * 128;
      // (features beyond the last have some scale of the matrix: they are not stored)
      const float* xs = a.x_scales + min(row, last - 1);
      const int block = a.pairs ? m.n_tile * 2 : min(m.n_tile * 2 + half, a.scale_rows - 1);
      const float* we = a.w_scales + ((size_t)m.expert * a.scale_rows + block) * a.runs;
      const float* wo = a.pairs ? we + a.runs : we;
      f32x2 sum[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) sum[c] = f2_pack(0.f, 0.f);
      // a step's scales are asked for two steps ahead, into the registers of the step before last (a move from one to the other would wait)
      float x[2], e[2], o[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = min(i, a.runs - 1);
        x[i] = xs[(size_t)at * a.lds]; e[i] = we[at]; o[i] = wo[at];
      }
      auto step = [&](int kb, int i) {
        outside |= a.far.outside(x[i]);
        const f32x2 scale = f2_pack(x[i] * e[i], x[i] * o[i]);
        const int at = min(kb + 2, a.runs - 1);
        x[i] = xs[(size_t)at * a.lds]; e[i] = we[at]; o[i] = wo[at];
        if (!mbar_wait_warp(acc_full_bar(b), acc_phase)) {
          if (a.error_word && lane == 0) atomicExch(a.error_word, 0x7C00D3);
          ok = false;
          return;
        }
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + b * 256 + half * 128;
        uint32_t v[2][16];
        tmem_ld16(acc, v[0]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
          if (c < 7) tmem_ld16(acc + 16 * (c + 1), v[(c + 1) & 1]);
          else {                               // read: tell the MMA warp (in the even block)
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) b2_arrive_even(map_to_cta(acc_empty_bar(b), 0));
          }
#pragma unroll
          for (int q = 0; q < 8; ++q)
            sum[8 * c + q] = f2_fma(f2_pack(__uint_as_float(v[c & 1][2 * q]), __uint_as_float(v[c & 1][2 * q + 1])), scale, sum[8 * c + q]);
        }
        if (++b == 2) { b = 0; acc_phase ^= 1; }
      };
#pragma unroll 1
      for (int kb = 0; kb < a.runs && ok; kb += 2) {
        step(kb, 0);
        if (kb + 1 < a.runs && ok) step(kb + 1, 1);
      }
      if (!ok) continue;
      if (a.ep.row_scale) {
        const float scale = a.ep.row_scale[bs_pair(a.order, min(row, last - 1), a.M)];
        const f32x2 scale2 = f2_pack(scale, scale);
#pragma unroll
        for (int c = 0; c < 64; ++c) sum[c] = f2_mul(sum[c], scale2);
      }
      // A row's outputs lie in one thread: a warp's 32 rows cross its 4 KB of shared memory, 128 bytes of each at a time (16-byte pieces, swizzled by row),
      // and leave as whole lines.  (Stored by their threads, 16 bytes of 32 rows an instruction, a tile's outputs took 3 us.)
      constexpr bool kGated = moe_act_gated(ACT);
      constexpr int kOut = kGated ? 64 : 128, kVec = 16 / sizeof(TO), kTurn = 8 * kVec;      // outputs of a thread, a piece, a turn
      const int first = col0 >> kGated, n_out = a.N >> kGated;
      unsigned char* mine = smem_raw + (base - smem_u32(smem_raw)) + kB2Stages * kB2Stage + 256 + (warp - 4) * 4096;
#pragma unroll
      for (int turn = 0; turn < kOut / kTurn; ++turn) {
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          float y[kVec];
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const int c = turn * kTurn + p * kVec + j;
            float lo, hi;
            f2_unpack(sum[kGated ? c : c >> 1], lo, hi);
            y[j] = kGated ? bs_gated<ACT>(lo, hi, a.ep.limit, a.ep.alpha) : bs_act<ACT>(c & 1 ? hi : lo);
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
              const TO v = *reinterpret_cast<const TO*>(mine + r * 128 + (((c / kVec) ^ (r & 7)) << 4) + (c % kVec) * sizeof(TO));
              const int col = first + turn * kTurn + c;
              if (col < n_out) out[(size_t)(row - lane + r) * ldo + col] = v;
            }
          }
        }
        __syncwarp();
      }
    }
    if (__any_sync(0xffffffffu, outside) && ok)      // (behind all tiles: among them it would take registers from their loop)
      for (int t = pair; t < num_tiles; t += pairs) {
        const B2Tile m = tile_of(t);
        const int row0 = (int)rank * 128 + quarter * 32;
        if (row0 < m.rows) b2_rows_apart<ACT>(&a, m.first + row0, min(32, m.rows - row0), m.expert, (m.n_tile * 256 + half * 128) >> moe_act_gated(ACT), out, ldo);
      }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n");
    if (warp == 0) {
      const uint32_t leader = umma_leader();
      int s = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += pairs) {
        const B2Tile m = tile_of(t);
        const int m0 = m.first + (int)rank * 128;          // (behind the tile's rows come others', which are not stored, or zeros)
        const int w_block = m.n_tile * 2 + (int)rank, blocks = (a.N + 127) >> 7;
        // (a pair's second block of features may lie behind the matrix: it reads some block of it instead, which is not stored)
        const int w0 = (m.expert * blocks + min(w_block, blocks - 1)) * a.runs;
        for (int kb = 0; kb < a.runs; ++kb) {
          if (!mbar_wait_warp(empty_bar(s), phase)) {
            if (a.error_word && leader) atomicExch(a.error_word, 0x7C00D1);
            ok = false;
            break;
          }
          if (leader) {
            if (rank == 0) mbar_expect_tx(full_bar(s), 2 * kB2Stage);
            const uint32_t bar0 = map_to_cta(full_bar(s), 0);
            pair_tma_load(base + s * kB2Stage, &map_x, kb * kBlk, m0, bar0);
            pair_tma_load(base + s * kB2Stage + kB2Half, &map_w, 0, (w0 + kb) << 7, bar0);
          }
          __syncwarp();
          if (++s == kB2Stages) { s = 0; phase ^= 1; }
        }
      }
      // The even block's last releases of the stages arrive here as well: they have come before this block leaves.
      for (int i = 0; i < kB2Stages && ok; ++i) {
        if (!mbar_wait_warp(empty_bar(s), phase)) {
          if (a.error_word && leader) atomicExch(a.error_word, 0x7C00D1);
          ok = false;
        }
        if (++s == kB2Stages) { s = 0; phase ^= 1; }
      }
    } else if (warp == 1) {
      if (rank == 0) {
        const uint32_t leader = umma_leader();
        int s = 0, b = 0;
        uint32_t phase = 0, acc_phase = 1;
        bool ok = true;
        for (int t = pair; t < num_tiles && ok; t += pairs) {
          for (int kb = 0; kb < a.runs; ++kb) {
            if (!__all_sync(0xffffffffu, pair_wait(full_bar(s), phase))) {
              if (a.error_word && leader) atomicExch(a.error_word, 0x7C00D2);
              ok = false;
              break;
            }
            if (!__all_sync(0xffffffffu, pair_wait(acc_empty_bar(b), acc_phase))) {      // both blocks have read this accumulator
              if (a.error_word && leader) atomicExch(a.error_word, 0x7C00D4);
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const uint32_t x_src = umma_low_k128(base + s * kB2Stage), w_src = x_src + (kB2Half >> 4);
  #pragma unroll
            for (int k = 0; k < 4; ++k) b2_umma(leader, tmem_base + b * 256, x_src + 2 * k, w_src + 2 * k, k != 0);
            if (leader) {
              pair_commit_both(acc_full_bar(b));
              pair_commit_both(empty_bar(s));      // the stage is free in both blocks once these MMAs have read it
            }
            __syncwarp();
            if (++s == kB2Stages) { s = 0; phase ^= 1; }
            if (++b == 2) { b = 0; acc_phase ^= 1; }
          }
        }
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

static int64_t b2_tiles(int M, int N, int experts) {      // at most; experts: 0 for one matrix
  return (int64_t)(experts ? M / 256 + (M < experts ? M : experts) : ceil_div(M, 256)) * ceil_div(N, 256);
}

template <int ACT, typename TO>
static int launch_b2(const CUtensorMap& map_x, const CUtensorMap& map_w, const B2Args& a, void* out, int64_t ldo, cudaStream_t stream) {
  auto kern = block_scaled_2cta_kernel<ACT, TO>;
  static bool allowed[64];      // (by device: the attribute belongs to its context)
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && !(device < 64 && allowed[device])) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
  if (e != cudaSuccess) return (int)e;
  if (device < 64) allowed[device] = true;
  const int64_t tiles = b2_tiles(a.M, a.N, a.offsets ? a.experts : 0);
  if (tiles > 0x7fffffff) return TIB_E_SIZE;
  const int wide = ((uintptr_t)out & 15) == 0 && (ldo * sizeof(TO)) % 16 == 0;
  TIB_LAUNCH_DEPENDENT(kern, 2 * (int)(tiles < 74 ? tiles : 74), kB2Threads, kB2Smem + (a.offsets ? 8 * (a.experts + 1) : 0), stream, map_x, map_w, a, (TO*)out,
                       ldo, wide);
  return TIB_OK;
}

}  // namespace tib

using namespace tib;

TIB_API int tib_block_scaled_2cta_experts() { return kB2MaxExperts; }

// See tib_block_scaled_plan.
TIB_API int tib_block_scaled_2cta_plan(int M, int N, int K, int experts, int* plan) {
  if (!plan || M < 1 || N < 1 || K < 1 || experts < 0 || experts > kB2MaxExperts) return TIB_E_ARG;
  const int64_t tiles = b2_tiles(M, N, experts), steps = ceil_div(K, kBlk) * ceil_div64(tiles, tiles < 74 ? tiles : 74);
  plan[0] = 256; plan[1] = 1; plan[2] = (int)(steps < 0x7fffffff ? steps : 0x7fffffff); plan[3] = kB2Stages;
  return TIB_OK;
}

// x: codes [M, runs * 128] and scales [runs, lds] as tib_quantize_rows leaves them; w: codes in blocks [experts, ceil(N / 128), runs, 128, 128] and
// scales [experts, scale_rows, runs] (`pairs`: of (gate, up) row pairs, N and scale_rows even); out: [M, N] in out_dtype (row stride ldo), or [M, N / 2] of a
// gated activation.  offsets [experts + 1] and order [M]: rows sorted by expert, at most kB2MaxExperts of them; offsets null: one matrix for all rows.
// far_low, far_high: see BsFar.
TIB_API int tib_block_scaled_2cta(const void* x, const float* x_scales, int64_t lds, const void* w, const float* w_scales, int scale_rows, int pairs,
                                  void* out, int out_dtype, int64_t ldo, int M, int N, int K, const int* offsets, const int* order, int experts, int act,
                                  float limit, float alpha, const float* row_scale, float far_low, float far_high, int* error_word, cudaStream_t stream) {
  if (M == 0 || N == 0) return TIB_OK;
  if (!x || !x_scales || !w || !w_scales || !out || M < 0 || N < 0 || K < 1 || scale_rows < 1 || experts < 1) return TIB_E_ARG;
  if ((offsets && !order) || (row_scale && !order)) return TIB_E_ARG;
  if (act < MOE_ACT_NONE || act > MOE_ACT_GELU || (moe_act_gated(act) && !pairs) || (pairs && (N % 2 || scale_rows % 2)) || lds < M) return TIB_E_SIZE;
  if (experts > kB2MaxExperts || (int64_t)experts * ceil_div(N, 128) * ceil_div(K, kBlk) > (0x7fffffff >> 7)) return TIB_E_SIZE;
  if (out_dtype != TIB_BF16 && out_dtype != TIB_F32) return TIB_E_DTYPE;
  if (((uintptr_t)x | (uintptr_t)w) & 15) return TIB_E_ALIGN;
  B2Args a;
  a.x = static_cast<const unsigned char*>(x); a.w = static_cast<const unsigned char*>(w); a.far = BsFar{far_low, far_high};
  a.x_scales = x_scales; a.lds = lds; a.w_scales = w_scales; a.scale_rows = scale_rows; a.pairs = pairs;
  a.M = M; a.N = N; a.runs = ceil_div(K, kBlk); a.offsets = offsets; a.order = order; a.experts = experts; a.error_word = error_word;
  a.ep.act = act; a.ep.limit = limit; a.ep.alpha = alpha; a.ep.row_scale = row_scale;
  CUtensorMap map_x, map_w;
  int rc = bs_make_map(&map_x, x, M, (int64_t)a.runs * kBlk, 128);
  if (rc != TIB_OK) return rc;
  rc = bs_make_map(&map_w, w, (int64_t)experts * ceil_div(N, 128) * a.runs * 128, kBlk, 128);
  if (rc != TIB_OK) return rc;
#define TIB_B2_GO(ACT) \
  case ACT: return out_dtype == TIB_BF16 ? launch_b2<ACT, __nv_bfloat16>(map_x, map_w, a, out, ldo, stream) : launch_b2<ACT, float>(map_x, map_w, a, out, ldo, stream)
  switch (act) {
    TIB_B2_GO(MOE_ACT_NONE);
    TIB_B2_GO(MOE_ACT_RELU2);
    TIB_B2_GO(MOE_ACT_SILU);
    TIB_B2_GO(MOE_ACT_GELU);
    TIB_B2_GO(MOE_ACT_GLU_CLAMP);
    TIB_B2_GO(MOE_ACT_SWIGLU);
  }
#undef TIB_B2_GO
  return TIB_E_SIZE;
}
