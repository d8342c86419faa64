// 8-bit integer product with a scale for each row and each channel (sm_100a).
//
//   y[m, n] = (sum_k xq[m, k] wq[n, k]) * sx[m] * sw[n] (+ bias[n])
//
// xq [rows, K], wq [n_out, K] int8, K-major; the sum is exact in the tensor cores' 32-bit
// integers (tcgen05 kind::i8), so no order of additions shows in the result.
//
// The weights are the MMA's M side (128 TMEM lanes, one channel each) and the rows its N
// side (TN columns), whatever the number of rows: a weight-streaming call of a few rows
// loads 128 channels for every TN = 16 rows, and a large call runs full 128 x 256 tiles.
// K goes in blocks of 128 (one 128-byte swizzled line of every operand row), staged by TMA
// in a ring; two accumulators in TMEM let a tile's epilogue overlap the next one's MMAs.
//
// Warp roles (224 threads): warps 0 and 6 = TMA producers (weights, rows), warp 1 = TMEM
// allocator + MMA issuer, warps 2..5 = epilogue (one thread per channel).  Two producers,
// because one copy takes about 150 cycles to issue: with both operands' on one warp a block of K
// took 335 cycles, now about 170.
//
// Bound by the weights' bytes at few rows: 16 x 151936 x 4096 (625 MB) 97 us, 6.4 TB/s, as
// a plain copy.  Small products are a chain of latencies (16 x 256 x 4096 8.4 us with the
// quantisation).  With more than 128 rows CTA pairs may share the tiles (i8_pair_kernel).
#pragma once

#include "tc_gemm.cuh"

namespace dels {

constexpr int kI8BK = 128;  // K elements (bytes) of a block
constexpr int kI8Threads = 224;

struct I8Args {
  int rows, n_out, kb;     // kb: blocks of K
  int box;                 // channels a weight tile loads (<= 128; the MMA always runs 128 lanes)
  int stages;              // of the ring
  int n_tiles, m_tiles;    // weight tiles, row tiles
  const float* sx;         // [rows]
  const float* sw;         // [n_out]
  const void* bias;        // [n_out] of the output's type, or null
  void* out;               // [rows, n_out] bf16 or fp32
  long long ld_out;
  int store2;              // bf16: two channels per store (even ld_out, 4-byte aligned out)
  int bn, tail;            // i8_pair_kernel: rows of a tile, ways one of the last wave is split along them
  int early;               // the weights are not written by the previous kernel: load them before waiting for it
  int* status;
};

constexpr int kI8MaxStages = 32;
constexpr int kI8MostCtas = 3;  // of an SM: 16 x 151936 x 64 in 9.1 us (2: 11.6, 4: 9.5)

// Shared memory: the barriers and the row scales, then the ring: args.stages weight slots of
// args.box lines, 16 KB for the lanes that the last of them leaves unloaded, the rows' slots.
// (An MMA always reads 128 lines: what it finds past a slot goes to lanes that nobody reads.)
template <int TN>
struct I8Config {
  static constexpr int kBBytes = TN * kI8BK;
  static constexpr int kTmemCols = 2 * TN;
  static constexpr int kNumBars = 2 * kI8MaxStages + 4;
  static constexpr int kScaleOffset = kNumBars * 8 + 16;                    // [4 warps][TN] row scales
  static constexpr int kFixedBytes = kScaleOffset + 4 * TN * 4 + 1024 + kBM * kI8BK;
  static constexpr int kMaxBytes = 224 * 1024;
  static constexpr int slot_bytes(int box) { return box * kI8BK + kBBytes; }
  // as many blocks of K in flight as fit: a small tile's whole K
  static constexpr int stages(int box, int kb) {
    const int fit = (kMaxBytes - kFixedBytes) / slot_bytes(box);
    const int most = fit < kI8MaxStages ? fit : kI8MaxStages;
    return kb < 2 ? 2 : (kb < most ? kb : most);
  }
  static_assert(TN >= 16 && TN <= 256 && (TN & (TN - 1)) == 0, "TN is a power of two in [16, 256]");
  static_assert(kFixedBytes + 4 * slot_bytes(kBM) <= kMaxBytes, "four stages of the largest tile fit");
};

// One lane of the (converged) warp.  Inside a branch on it the compiler knows that one thread
// runs: the copies and MMAs there take their operands from uniform registers at once, where a
// branch on lane == 0 costs several hundred cycles for each block of K.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(one));
  return one != 0;
}

// D[tmem] (+)= A[smem] * B[smem]^T, signed 8-bit inputs, 32-bit integer accumulator.
__device__ __forceinline__ void tc_mma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor of tcgen05.mma kind::i8: signed A and B (both K-major), s32
// accumulator, shape M x N.
__host__ __device__ constexpr uint32_t make_idesc_s8_s32(int M, int N) {
  return (2u << 4)                        // accumulator format: s32
         | (1u << 7)                      // A format: signed
         | (1u << 10)                     // B format: signed
         | ((uint32_t)(N >> 3) << 17)     // N / 8
         | ((uint32_t)(M >> 4) << 24);    // M / 16
}

// A result from its integer sum: two roundings of the product, the second with the bias (0 where
// there is none), the same in every kernel, so that a row's results do not depend on its company.
__device__ __forceinline__ float i8_result(int sum, float sx, float sw, float bias) {
  return __fmaf_rn(__fmul_rn(__int2float_rn(sum), sx), sw, bias);
}

// One channel's results for the COLS rows row0.. of a tile; `valid` of them exist, the others
// are computed all the same and not stored, so that no branch keeps the rows' chains apart.
template <int COLS, typename OutT>
__device__ __forceinline__ void i8_store(const uint32_t (&v)[COLS], const float* scale, float sw, float bias, int valid,
                                         bool channel_ok, OutT* out, long long ld, bool store2, int lane) {
  if constexpr (sizeof(OutT) == 2) {
    if (store2) {
      // lanes 2i and 2i + 1 swap halves of a pair of rows, so each stores two neighbouring
      // channels of one row with one 4-byte store
      const bool odd = lane & 1;
#pragma unroll
      for (int j = 0; j < COLS; j += 2) {
        const float y0 = i8_result((int)v[j], scale[j], sw, bias);
        const float y1 = i8_result((int)v[j + 1], scale[j + 1], sw, bias);
        const float other = __shfl_xor_sync(0xffffffffu, odd ? y0 : y1, 1);
        const uint32_t pair = odd ? pack_bf16x2(other, y1) : pack_bf16x2(y0, other);
        if (channel_ok && j + (int)odd < valid)
          *reinterpret_cast<uint32_t*>(out + (long long)(j + (int)odd) * ld - (int)odd) = pair;
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    const float y = i8_result((int)v[j], scale[j], sw, bias);
    if (channel_ok && j < valid) {
      if constexpr (sizeof(OutT) == 2)
        out[j * ld] = __float2bfloat16_rn(y);
      else
        out[j * ld] = y;
    }
  }
}

template <int TN, typename OutT>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const I8Args args) {
  using Cfg = I8Config<TN>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int S = args.stages;
  const uint32_t a_bytes = (uint32_t)args.box * kI8BK;  // eight lines (1 KB) are a swizzle atom
  const uint32_t a_base = (smem_u32(smem) + (uint32_t)(Cfg::kScaleOffset + 4 * TN * 4) + 1023u) & ~1023u;
  const uint32_t b_base = a_base + S * a_bytes + kBM * kI8BK;
  float* scales = reinterpret_cast<float*>(smem + Cfg::kScaleOffset);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  auto full_bar = [&](int s) { return smem_u32(&bars[s]); };
  auto empty_bar = [&](int s) { return smem_u32(&bars[S + s]); };
  auto tfull_bar = [&](int a) { return smem_u32(&bars[2 * S + a]); };
  auto tempty_bar = [&](int a) { return smem_u32(&bars[2 * S + 2 + a]); };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 2);  // the weights' and the rows' producer
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int units = args.n_tiles * args.m_tiles;  // row tiles of one weight tile next to each other

  if (warp == 0 || warp == 6) {
    // ---------------------------------------------------------------- TMA producers
    // One warp for the weights and one for the rows: issuing a copy takes about as long as the
    // MMAs of half a narrow tile's block.  The weights need not wait for the kernel before.
    if (elect_one()) {
      const bool weights = warp == 0;
      const uint32_t bytes = weights ? a_bytes : (uint32_t)Cfg::kBBytes;
      const uint32_t ring = weights ? a_base : b_base;
      const CUtensorMap* map = weights ? &map_w : &map_x;
      if (!weights || !args.early) pdl_wait();
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const int y = weights ? u / args.m_tiles * args.box : u % args.m_tiles * TN;
        for (int kb = 0; kb < args.kb; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, args.status)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full_bar(stage), bytes);
          tma_load_2d(ring + stage * bytes, map, full_bar(stage), kb * kI8BK, y);
          ++issued;
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        // Aborting: let the copies already in flight land before the CTA exits (their stages
        // may lack the other producer's part: the wait is bounded).
        const int outstanding = issued < S ? issued : S;
        const unsigned long long t0 = globaltimer_ns();
        for (int i = 0; i < outstanding; ++i) {
          if (--stage < 0) {
            stage = S - 1;
            phase ^= 1u;
          }
          while (!mbar_try_wait(full_bar(stage), phase) && globaltimer_ns() - t0 < kWaitLimitNs / 20) {
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_s8_s32(kBM, TN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, args.status)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * TN);
        for (int kb = 0; kb < args.kb; ++kb) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag, args.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t adesc = make_sw128_desc(a_base + stage * a_bytes);
          const uint64_t bdesc = make_sw128_desc(b_base + stage * Cfg::kBBytes);
#pragma unroll
          for (int k = 0; k < kI8BK / 32; ++k)  // +32 bytes per K step inside the 128-byte swizzled line
            tc_mma_i8(d_tmem, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc, (kb > 0 || k > 0) ? 1u : 0u);
          tc_commit(empty_bar(stage));
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
        tc_commit(tfull_bar(acc));
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      // Aborting: wait until every MMA issued has completed before TMEM is released.
      if (!ok || *abort_flag) {
        const uint32_t drain = tfull_bar(acc);
        tc_commit(drain);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, acc_phase) && globaltimer_ns() - t0 < kWaitLimitNs / 20) {
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    pdl_wait();  // sx is another kernel's, and out may be in its hands
    const int quad = warp & 3;  // TMEM lanes this warp can read
    float* scale = scales + quad * TN;
    OutT* out = static_cast<OutT*>(args.out);
    const OutT* bias_v = static_cast<const OutT*>(args.bias);
    int acc = 0, scale_m = -1;
    uint32_t acc_phase = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const int m_tile = u % args.m_tiles, m0 = m_tile * TN;
      const int in_tile = quad * 32 + lane;
      const int n = u / args.m_tiles * args.box + in_tile;
      const bool channel_ok = in_tile < args.box && n < args.n_out;
      const bool warp_ok = quad * 32 < args.box && n - lane < args.n_out;
      const int valid = min(TN, args.rows - m0);
      if (m_tile != scale_m) {
        __syncwarp();
        for (int j = lane; j < TN; j += 32) scale[j] = m0 + j < args.rows ? args.sx[m0 + j] : 0.0f;
        __syncwarp();
        scale_m = m_tile;
      }
      const float sw = channel_ok ? args.sw[n] : 0.0f;
      float bias = 0.0f;
      if (channel_ok && bias_v != nullptr) {
        if constexpr (sizeof(OutT) == 2)
          bias = __bfloat162float(bias_v[n]);
        else
          bias = bias_v[n];
      }
      if (!mbar_wait(tfull_bar(acc), acc_phase, abort_flag, args.status)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * TN);
      OutT* dst = out + (long long)m0 * args.ld_out + n;
      if (warp_ok) {
        if constexpr (TN == 16) {
          uint32_t v[16];
          tmem_ld_16cols(t_row, v);
          tmem_ld_wait(v);
          i8_store<16, OutT>(v, scale, sw, bias, valid, channel_ok, dst, args.ld_out, args.store2 != 0, lane);
        } else {
#pragma unroll 1
          for (int c = 0; c < TN && c < valid; c += 32) {
            uint32_t v[32];
            tmem_ld_32cols(t_row + (uint32_t)c, v);
            tmem_ld_wait(v);
            i8_store<32, OutT>(v, scale + c, sw, bias, valid - c, channel_ok, dst + (long long)c * args.ld_out,
                               args.ld_out, args.store2 != 0, lane);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty_bar(acc));
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

// --------------------------------------------------------------------------------
// The same product on CTA pairs (tcgen05.mma.cta_group::2), for more than 128 rows: a tile is
// 256 channels x up to 256 rows (a multiple of 32 that the rows fill well), each CTA stages its
// 128 channels and half of the rows' tile, so a block of K moves 32 KB through each SM's shared
// memory for the work that takes 48 KB in i8_gemm_kernel.  The barriers are those of
// tc_scorer_pair_kernel: rank 0 issues the MMAs of both CTAs, whose copies complete on rank 0's
// full barriers.  Two blocks of K form a stage (256 contiguous bytes of every channel).  The
// last, partial wave's tiles are split along the rows (make_schedule's tail).
//
// Bound by the tensor cores and the board's power: 512 x 151936 x 4096 (637 G operations) 217 us
// at 1.58 GHz with the tensor pipe active 83 % of the cycles, 231-284 us (2.2-2.8 P operations a
// second) in longer runs, where the clock falls under the power cap.
// --------------------------------------------------------------------------------
struct I8PairConfig {
  static constexpr int BN = 256;                 // most rows of a tile
  static constexpr int kGroup = 2;               // blocks of K in a stage
  static constexpr int kABytes = kBM * kI8BK;
  static constexpr int kBBytes = BN / 2 * kI8BK;
  static constexpr int kSlots = 6;
  static constexpr int kStages = kSlots / kGroup;
  static constexpr int kScaleOffset = kSlots * (kABytes + kBBytes);  // [4 warps][BN] row scales
  static constexpr int kBarOffset = kScaleOffset + 4 * BN * 4;
  static constexpr int kNumBars = 2 * kStages + 4;
  static constexpr int kSmemBytes = kBarOffset + kNumBars * 8 + 16 + 1024;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

__device__ __forceinline__ void tc_mma_pair_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// map_x / map_xt: the rows in boxes of 128 and of 128 / args.tail (a split tile's half).
template <typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTcThreads, 1)
    i8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ CUtensorMap map_xt, const I8Args args) {
  using Cfg = I8PairConfig;
  constexpr int S = Cfg::kStages, KG = Cfg::kGroup;
  const int BN = args.bn;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base_addr = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base_addr - raw_addr);
  const uint32_t a_base = base_addr;
  const uint32_t b_base = base_addr + Cfg::kSlots * Cfg::kABytes;
  float* scales = reinterpret_cast<float*>(smem + Cfg::kScaleOffset);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOffset);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  auto full_bar = [&](int s) { return smem_u32(&bars[s]); };
  auto empty_bar = [&](int s) { return smem_u32(&bars[S + s]); };
  auto tfull_bar = [&](int a) { return smem_u32(&bars[2 * S + a]); };
  auto tempty_bar = [&](int a) { return smem_u32(&bars[2 * S + 2 + a]); };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 8);  // 4 epilogue warps in each CTA
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_xt);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers are initialised
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  // "columns" of the schedule are row tiles, its "row tiles" the weight tiles of this product:
  // neighbouring units share a weight tile
  const Schedule sched = make_schedule(args.m_tiles, args.n_tiles, 1, args.m_tiles, args.tail, num_pairs);
  // a unit: weight tile, first row, rows (BN or a split tile's)
  auto unit = [&](int u, int& n_tile, int& m0, int& rows, bool& tail) {
    tail = u >= sched.main_units;
    const int q = u - sched.main_units;
    const int t = tail ? sched.main_units + q / sched.tail_split : u;
    n_tile = t / args.m_tiles;
    rows = tail ? BN / sched.tail_split : BN;
    m0 = t % args.m_tiles * BN + (tail ? q % sched.tail_split * rows : 0);
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer (both CTAs)
    if (elect_one()) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = pair; u < sched.total_units && ok; u += num_pairs) {
        int n_tile, m0, rows;
        bool tail;
        unit(u, n_tile, m0, rows, tail);
        const int n0 = n_tile * 2 * kBM + (int)rank * kBM, x0 = m0 + (int)rank * (rows / 2);
        const CUtensorMap* mx = tail ? &map_xt : &map_x;
        const uint32_t tx_pair = 2u * ((uint32_t)Cfg::kABytes + (uint32_t)(rows / 2) * kI8BK);
        for (int kb = 0; kb < args.kb; kb += KG) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, args.status)) {
            ok = false;
            break;
          }
          const int nb = args.kb - kb < KG ? args.kb - kb : KG;
          const uint32_t full_leader = mapa_shared(full_bar(stage), 0);
          if (leader) mbar_arrive_expect_tx(full_bar(stage), tx_pair * (uint32_t)nb);
          for (int j = 0; j < nb; ++j) {
            const int slot = stage * KG + j, k = (kb + j) * kI8BK;
            tma_load_2d_pair(a_base + slot * Cfg::kABytes, &map_w, full_leader, k, n0);
            tma_load_2d_pair(b_base + slot * Cfg::kBBytes, mx, full_leader, k, x0);
          }
          ++issued;
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        // Aborting: the copies in flight complete on rank 0's full barriers; rank 0 drains
        // them, the peer waits out the same bounded delay before leaving.
        const unsigned long long t0 = globaltimer_ns();
        const int outstanding = issued < S ? issued : S;
        for (int i = 0; i < outstanding && leader; ++i) {
          if (--stage < 0) {
            stage = S - 1;
            phase ^= 1u;
          }
          while (!mbar_try_wait(full_bar(stage), phase) && globaltimer_ns() - t0 < kWaitLimitNs / 20) {
          }
        }
        while (!leader && globaltimer_ns() - t0 < kWaitLimitNs / 40) {
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (rank 0)
    if (leader && elect_one()) {
      const uint32_t idesc_full = make_idesc_s8_s32(2 * kBM, BN);
      const uint32_t idesc_tail = make_idesc_s8_s32(2 * kBM, BN / sched.tail_split);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int u = pair; u < sched.total_units && ok; u += num_pairs) {
        const uint32_t idesc = u >= sched.main_units ? idesc_tail : idesc_full;
        if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, args.status)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * Cfg::BN);
        for (int kb = 0; kb < args.kb; kb += KG) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag, args.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int nb = args.kb - kb < KG ? args.kb - kb : KG;
          for (int j = 0; j < nb; ++j) {
            const int slot = stage * KG + j;
            const uint64_t adesc = make_sw128_desc(a_base + slot * Cfg::kABytes);
            const uint64_t bdesc = make_sw128_desc(b_base + slot * Cfg::kBBytes);
#pragma unroll
            for (int k = 0; k < kI8BK / 32; ++k)
              tc_mma_pair_i8(d_tmem, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc,
                             (kb + j > 0 || k > 0) ? 1u : 0u);
          }
          tc_commit_pair_both(empty_bar(stage));
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
        tc_commit_pair_both(tfull_bar(acc));
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok || *abort_flag) {
        const uint32_t drain = tfull_bar(acc);
        tc_commit_pair_both(drain);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, acc_phase) && globaltimer_ns() - t0 < kWaitLimitNs / 20) {
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue (both CTAs)
    const int quad = warp & 3;
    float* scale = scales + quad * Cfg::BN;
    const uint32_t tempty_leader0 = mapa_shared(tempty_bar(0), 0);
    const uint32_t tempty_leader1 = mapa_shared(tempty_bar(1), 0);
    OutT* out = static_cast<OutT*>(args.out);
    const OutT* bias_v = static_cast<const OutT*>(args.bias);
    int acc = 0, scale_m = -1;
    uint32_t acc_phase = 0;
    for (int u = pair; u < sched.total_units; u += num_pairs) {
      int n_tile, m0, rows;
      bool tail;
      unit(u, n_tile, m0, rows, tail);
      const int n = n_tile * 2 * kBM + (int)rank * kBM + quad * 32 + lane;
      const bool channel_ok = n < args.n_out, warp_ok = n - lane < args.n_out;
      const int valid = min(rows, args.rows - m0);  // may be <= 0 in a split tile
      if (m0 != scale_m) {
        __syncwarp();
        for (int j = lane; j < rows; j += 32) scale[j] = m0 + j < args.rows ? args.sx[m0 + j] : 0.0f;
        __syncwarp();
        scale_m = m0;
      }
      const float sw = channel_ok ? args.sw[n] : 0.0f;
      float bias = 0.0f;
      if (channel_ok && bias_v != nullptr) {
        if constexpr (sizeof(OutT) == 2)
          bias = __bfloat162float(bias_v[n]);
        else
          bias = bias_v[n];
      }
      if (!mbar_wait(tfull_bar(acc), acc_phase, abort_flag, args.status)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * Cfg::BN);
      OutT* dst = out + (long long)m0 * args.ld_out + n;
#pragma unroll 1
      for (int c = 0; c < (warp_ok ? valid : 0); c += 32) {
        uint32_t v[32];
        tmem_ld_32cols(t_row + (uint32_t)c, v);
        tmem_ld_wait(v);
        i8_store<32, OutT>(v, scale + c, sw, bias, valid - c, channel_ok, dst + (long long)c * args.ld_out, args.ld_out,
                           args.store2 != 0, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader)
          mbar_arrive(tempty_bar(acc));
        else
          mbar_arrive_remote(acc == 0 ? tempty_leader0 : tempty_leader1);
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the partner no longer touches this CTA's shared memory / TMEM
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// Rows to 8 bits (i8_kernels.cu): scale = max |x| / 127, q = rint(x * (127 / max |x|)).
constexpr int kQuantThreads = 256;
using QuantizeKernel = void (*)(const void* x, long long ld_x, int rows, int K, int8_t* q, long long ld_q, float* scale);
// for bf16 or fp32 rows, with 16-byte loads (vec) or without
QuantizeKernel quantize_rows_kernel_for(bool bf16, bool vec);

// A few rows against all channels in one launch: each CTA quantises the rows for itself (or
// copies quantised ones) into shared memory, then a warp takes one, two or four channels at a
// time with dp4a (i8_kernels.cu).
constexpr int kI8GemvThreads = 256;
constexpr int kI8GemvCtas = 3;           // of an SM
constexpr int kI8GemvLoads = 8;          // 16-byte loads of a lane in flight
constexpr int kI8GemvRows = 2;           // most rows
constexpr int kI8GemvBytes = 32768;      // most bytes of quantised rows (an SM's CTAs hold them each)
enum I8Source { kI8FromInt8 = 0, kI8FromBf16 = 1, kI8FromF32 = 2 };
struct I8GemvArgs {
  const void* x;        // [rows, K], row stride ld_x elements
  long long ld_x;
  int vec;              // 16-byte loads of x
  const float* sx;      // [rows], with int8 rows
  const int8_t* w;
  long long ld_w;
  const float* sw;
  const void* bias;
  void* out;
  long long ld_out;
  int rows, K, n_out;
};
using I8GemvKernel = void (*)(I8GemvArgs);
I8GemvKernel i8_gemv_kernel_for(I8Source source, bool out_bf16, int rows, int channels);

}  // namespace dels
