// Beam drafting kernels.
//
// Selection.  A row is one beam's logits over the vocabulary, x[v] = logits[v], or
// x[v] = (base[v] + logits[v]) - beta prior[v] when the sequence's beams share draft logits
// and a prior.  A candidate (beam, v) scores
//
//   (x[v] - m) + (cum - log S)      m = max_v x[v],  S = sum_v exp(x[v] - m)
//
// which is cum + log_softmax(x)[v], written so that logits at the type's lowest value
// (masks) cancel before they meet anything small.  The best `select` candidates of a
// sequence: higher score, then lower beam, then larger x, then lower token.
//
//   beam_scan_kernel    one pass over the logits: per slice of a row the running (m, S) of
//                       an online softmax, and for every 512 logits the maxima of their four
//                       quarters.
//   beam_finish_kernel  a CTA per sequence.  The `select`-th largest score of those maxima, over
//                       all beams, bounds the sequence's `select` best scores from below, so
//                       only the quarters that reach it are read again.
//
// Both kernels are short loops on purpose: a step of one sequence runs each instruction a
// few times only, and then fetching code costs more than executing it (unrolled over four
// rows, the scan of 4 x 151936 logits took 23 us for 810 instructions a warp).
//
// A kernel here may start before the one that makes its inputs has ended (programmatic
// dependent launch), so nothing is read through the read-only path.
#include "beam_kernels.cuh"

namespace dels {

namespace {

constexpr uint32_t kAllLanes = 0xffffffffu;

__device__ __forceinline__ float neg_inf() { return -__int_as_float(0x7f800000); }

// Unsigned order of float order: NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t ordered_u32(float f) { return (uint32_t)ordered_i32_dev(f) ^ 0x80000000u; }
__device__ __forceinline__ float ordered_u32_to_float(uint32_t u) { return ordered_to_float((int32_t)(u ^ 0x80000000u)); }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// Warp maximum that is NaN when any lane's is.
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// 2^x by the special-function unit (relative error of 2^-22).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two packed fp32 additions or products in one instruction, each rounded by itself.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}

// a b + c of packed fp32, each rounded once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}

// (m, s) of two parts of a softmax; s counts exp(x - m).
__device__ __forceinline__ float2 softmax_join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  // a part without any finite logit has s = 0 (or NaN) and may have m = -inf
  const float ea = a.x == m ? 1.0f : __expf(a.x - m);
  const float eb = b.x == m ? 1.0f : __expf(b.x - m);
  return make_float2(m, a.y * ea + b.y * eb);
}

// ------------------------------------------------------------------ logits
// A lane's kPer logits of a group.  VEC (16-byte loads: rows aligned to 16 bytes, V a
// multiple of 8): two runs of eight, run h of lane l at 256 h + 8 l.  Otherwise every 32nd.
constexpr int kPer = kBeamGroup / 32;

// Quarter q of a group is the lanes' logits 4 q .. 4 q + 3; their offsets in the group.
template <bool VEC>
__device__ __forceinline__ int quarter_offset(int q, int lane, int j) {
  return VEC ? (q >> 1) * 256 + lane * 8 + (q & 1) * 4 + j : (4 * q + j) * 32 + lane;
}

// Four logits of a lane as they are loaded.
template <typename T>
struct Raw4;
template <>
struct Raw4<float> {
  float4 w;
  __device__ __forceinline__ void load(const float* p) {
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(w.x), "=f"(w.y), "=f"(w.z), "=f"(w.w)
                 : "l"(p));
  }
  __device__ __forceinline__ void unpack(float2 (&x)[2]) const { x[0] = make_float2(w.x, w.y), x[1] = make_float2(w.z, w.w); }
};
template <>
struct Raw4<__nv_bfloat16> {
  uint2 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "l"(p));
  }
  __device__ __forceinline__ void unpack(float2 (&x)[2]) const {
    x[0] = make_float2(bf16_lo(w.x), bf16_hi(w.x)), x[1] = make_float2(bf16_lo(w.y), bf16_hi(w.y));
  }
};

// A lane's logits of a group from their staged copy.
__device__ __forceinline__ void staged(const float* group, int lane, float2 (&x)[kPer / 2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 w = *reinterpret_cast<const float4*>(group + (i >> 1) * 256 + lane * 8 + (i & 1) * 4);
    x[2 * i] = make_float2(w.x, w.y), x[2 * i + 1] = make_float2(w.z, w.w);
  }
}
__device__ __forceinline__ void staged(const __nv_bfloat16* group, int lane, float2 (&x)[kPer / 2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 w = *reinterpret_cast<const uint4*>(group + h * 256 + lane * 8);
    x[4 * h] = make_float2(bf16_lo(w.x), bf16_hi(w.x)), x[4 * h + 1] = make_float2(bf16_lo(w.y), bf16_hi(w.y));
    x[4 * h + 2] = make_float2(bf16_lo(w.z), bf16_hi(w.z)), x[4 * h + 3] = make_float2(bf16_lo(w.w), bf16_hi(w.w));
  }
}

// Starts the copy of `bytes` (a multiple of 16) to shared memory, counted on `bar`.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// The draft logits and prior that a sequence's beams share; either may be missing.
template <typename T>
struct Shared {
  const T* base;
  const float* prior;
  float nbeta;  // -beta
};

template <typename T>
__device__ __forceinline__ Shared<T> shared_terms(const BeamSelectArgs& a, int seq) {
  Shared<T> sh{nullptr, nullptr, 0.0f};
  if (a.base != nullptr) sh.base = static_cast<const T*>(a.base) + (long long)seq * a.ld_base;
  if (a.prior != nullptr) sh.prior = a.prior, sh.nbeta = -*a.beta;
  return sh;
}

// x = (base + logit) - beta prior, every operation rounded by itself.
template <typename T>
__device__ __forceinline__ float mixed_logit(const T* row, const Shared<T>& sh, int v) {
  float x = to_f32(row[v]);
  if (sh.base != nullptr) x = __fadd_rn(to_f32(sh.base[v]), x);
  if (sh.prior != nullptr) x = __fadd_rn(x, __fmul_rn(sh.nbeta, sh.prior[v]));
  return x;
}

// A lane's logits of the group at v0 of two rows without 16-byte loads; -inf past V.  In a
// whole group all loads leave before the first of them is used.
template <typename T>
__device__ __forceinline__ void load_single(const T* const (&row)[2], const Shared<T>& sh, int v0, int V, int lane,
                                            float2 (&x)[2][kPer / 2]) {
  if (v0 + kBeamGroup <= V) {
    T w[2][kPer], b[kPer];
    float p[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int v = v0 + 32 * j + lane;
      w[0][j] = row[0][v], w[1][j] = row[1][v];
    }
    if (sh.base != nullptr) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) b[j] = sh.base[v0 + 32 * j + lane];
    }
    if (sh.prior != nullptr) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) p[j] = sh.prior[v0 + 32 * j + lane];
    }
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        x[r][i] = make_float2(to_f32(w[r][2 * i]), to_f32(w[r][2 * i + 1]));
        if (sh.base != nullptr) x[r][i] = add2(make_float2(to_f32(b[2 * i]), to_f32(b[2 * i + 1])), x[r][i]);
        if (sh.prior != nullptr)
          x[r][i] = add2(x[r][i], mul2(make_float2(sh.nbeta, sh.nbeta), make_float2(p[2 * i], p[2 * i + 1])));
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i) {
    const int u = v0 + 64 * i + lane, v = u + 32;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      x[r][i].x = u < V ? mixed_logit<T>(row[r], sh, u) : neg_inf();
      x[r][i].y = v < V ? mixed_logit<T>(row[r], sh, v) : neg_inf();
    }
  }
}

// The softmax of a warp's two rows as its run over them goes on.  nref: minus the reference of the
// exponentials (0 before there is one), the same in all lanes; (s.x, s.y): the lane's own sums of
// exp(x + nref) of the two, (less.x, less.y): what their rounding left out, to be added; m: lane
// r's maximum of row r.  A reference follows its maximum only when that passes `limit`, kLag above
// the reference: a row that climbs a little in every group would else be rounded by a rescaling in
// each.
struct RowSoftmax {
  float m, nref[2], limit[2];
  float2 s, less;
};
constexpr float kLag = 16.0f;

// Takes a lane's logits of a group of two rows into their running softmax; t: the maxima of the
// quarters, NaN where one holds it, and then the sums are NaN.  Two rows at a time fill each
// other's waits.  A group's terms are added in pairs and then, compensated, to the sum: one by one
// they rounded the same way, 5e-5 of a sum over 524288 equal logits.
__device__ __forceinline__ void fold_group(const float2 (&x)[2][kPer / 2], int lane, RowSoftmax& w, float4 (&t)[2]) {
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = fmax_nan(fmax3_nan(x[r][2 * i].x, x[r][2 * i].y, x[r][2 * i + 1].x), x[r][2 * i + 1].y);
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = warp_max_nan(q[i]);
    t[r] = make_float4(q[0], q[1], q[2], q[3]);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float top = fmax3_nan(fmax_nan(t[r].x, t[r].y), t[r].z, t[r].w);
    if (lane == r) w.m = fmaxf(w.m, top);
    if (top > w.limit[r]) {
      const float down = w.limit[r] == neg_inf() ? 0.0f : expf(-w.nref[r] - top);  // (the first one's sums are 0)
      const float2 by = r == 0 ? make_float2(down, 1.0f) : make_float2(1.0f, down);
      w.s = mul2(w.s, by);
      w.less = mul2(w.less, by);
      w.nref[r] = -top;
      w.limit[r] = top + kLag;
    }
  }
  float2 e[2][kPer / 2];
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float2 y =
          mul2(add2(x[r][i], make_float2(w.nref[r], w.nref[r])), make_float2(1.4426950408889634f, 1.4426950408889634f));
      e[r][i] = make_float2(exp2_approx(y.x), exp2_approx(y.y));
      // a pair is added as soon as both of its sums are there
#pragma unroll
      for (int o = 1; o < kPer / 2; o *= 2)
        if ((i & (2 * o - 1)) == 2 * o - 1) e[r][i] = add2(e[r][i - o], e[r][i]);
    }
  constexpr int last = kPer / 2 - 1;
  const float2 y = add2(make_float2(e[0][last].x + e[0][last].y, e[1][last].x + e[1][last].y), w.less);
  const float2 sum = add2(w.s, y);
  w.less = add2(y, fma2(sum, make_float2(-1.0f, -1.0f), w.s));
  w.s = sum;
}

}  // namespace

// ------------------------------------------------------------------ the scan
// A block is up to kBeamScanRows rows, of one sequence where its beams share draft logits or a
// prior, which they then meet in one CTA.  A team of warps scans a group, two rows a warp; the
// teams of a CTA take turns at the groups of its run: of one block, or of the end of one and the
// start of the next.  Each row's (m, S) of a CTA's share goes to part[row][CTA - first CTA of
// the block].  With VEC a team has the next groups copied into its ring in shared memory ahead
// of its arithmetic (bulk copies: no registers held, a handful of instructions a group).
//
// 64 x 8 beams of 151936 bf16 logits with shared ones, 175 MB: 49 us, 3.6 TB/s.  No unit is
// full (ALU pipe 39 %, FMA 37 %, special functions 41 %, 0.61 instructions a cycle of each
// scheduler): 398 instructions a warp and group, of which 32 are exponentials and 8 warp
// reductions, wait for one another, and 24 warps an SM hide a part of it.  Rows that cannot be
// copied (VEC false: 16-byte alignment, V a multiple of 8) are loaded a group at once instead:
// 64 x 8 beams without shared logits 63 us at an odd address, 48 us aligned; 1 x 4 beams 15.6
// and 11.2 us.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kBeamScanWarps, kBeamScanCtas) beam_scan_kernel(BeamSelectArgs a) {
  constexpr int D = beam_scan_depth(sizeof(T));
  constexpr int N = 2;  // rows of a warp
  extern __shared__ __align__(16) char smem[];
  __shared__ float2 team_part[kBeamScanWarps][kBeamScanRows];
  __shared__ uint64_t full[kBeamScanWarps][D], empty[kBeamScanWarps][D];  // [team][slot]
  __shared__ int aborted;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pairs = scan_pairs(a.scan_rows), teams = (blockDim.x >> 5) / pairs;
  const int team = warp / pairs, pair = warp % pairs;
  const int run_blocks = (a.run_rows + a.scan_rows - 1) / a.scan_rows;
  int unit = a.share.first(blockIdx.x);
  const int unit_end = a.share.first(blockIdx.x + 1);
  char* ring = smem + team * D * a.slot_bytes;
  if (VEC && threadIdx.x < kBeamScanWarps * D) {
    mbar_init(smem_u32(&full[0][0] + threadIdx.x), 1);
    mbar_init(smem_u32(&empty[0][0] + threadIdx.x), pairs);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) aborted = 0;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  int slot = 0, fill_slot = 0;
  uint32_t parity = 0, fill_parity = 0;
#pragma unroll 1
  while (unit < unit_end) {
    const int block = unit / a.groups, g_begin = unit - block * a.groups;
    const int g_end = min(a.groups, g_begin + (unit_end - unit));
    unit += g_end - g_begin;
    const int run = block / run_blocks;
    const int row0 = run * a.run_rows + block % run_blocks * a.scan_rows;
    const int n_rows = min(a.scan_rows, (run + 1) * a.run_rows - row0);
    const T* logits = static_cast<const T*>(a.logits) + (long long)row0 * a.ld;
    // the rows to scan: lane i < n_live holds the i-th one
    const bool mine = lane < n_rows && (a.finished == nullptr || a.finished[row0 + lane] == 0);
    const uint32_t live = __ballot_sync(kAllLanes, mine);
    const int n_live = __popc(live);
    if (n_live == 0) continue;
    int my_row = lane;
    if (n_live < n_rows) {
#pragma unroll 1
      for (int r = 0; r < n_rows; ++r)
        if (((live >> r) & 1u) && __popc(live & ((1u << r) - 1u)) == lane) my_row = r;
    }
    const int n_mine = min(N, n_live - N * pair);  // rows of this warp, from the N pair-th on
    const Shared<T> sh = shared_terms<T>(a, run);  // (without shared terms there is one run)
    RowSoftmax w = {neg_inf(), {0.0f, 0.0f}, {neg_inf(), neg_inf()}, {0.0f, 0.0f}, {0.0f, 0.0f}};
    float4* tops[N];
    const T* row[N];
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const int k = __shfl_sync(kAllLanes, my_row, min(N * pair + r, n_live - 1));
      tops[r] = a.ws.group_top + (long long)(row0 + k) * a.groups;
      row[r] = logits + k * a.ld;
    }
    // Lane i < n_live of the team's first warp copies the i-th row's part of a group into a
    // slot, the next two lanes those of the draft logits and the prior.
    const char* src = nullptr;
    uint32_t src_elem = sizeof(T);
    if (lane < n_live) src = reinterpret_cast<const char*>(logits + my_row * a.ld);
    if (lane == n_live && sh.base != nullptr) src = reinterpret_cast<const char*>(sh.base);
    if (lane == n_live + 1 && sh.prior != nullptr) src = reinterpret_cast<const char*>(sh.prior), src_elem = 4;
    const uint32_t token_bytes = __reduce_add_sync(kAllLanes, src != nullptr ? src_elem : 0u);
    const uint32_t dst = smem_u32(ring) + lane * kBeamGroup * sizeof(T);
    auto copy = [&](int k) {
      if (pair != 0 || k >= g_end) return;
      // a wait that gives up leaves its mark in the status word; the CTA then runs through
      mbar_wait(smem_u32(&empty[team][fill_slot]), fill_parity ^ 1u, &aborted, a.status);
      const uint32_t len = min(kBeamGroup, a.V - k * kBeamGroup), bar = smem_u32(&full[team][fill_slot]);
      if (lane == 0) mbar_arrive_expect_tx(bar, len * token_bytes);
      __syncwarp();
      if (src != nullptr)
        bulk_copy(dst + fill_slot * a.slot_bytes, src + (long long)k * kBeamGroup * src_elem, len * src_elem, bar);
      if (++fill_slot == D) fill_slot = 0, fill_parity ^= 1u;
    };
    int g = g_begin + team;
    if (VEC) {
#pragma unroll 1
      for (int i = 0; i < D - 1; ++i) copy(g + i * teams);
    }
#pragma unroll 1
    for (; g < g_end; g += teams) {
      const T* p = reinterpret_cast<const T*>(ring + slot * a.slot_bytes);
      const uint32_t read = smem_u32(&empty[team][slot]);
      if constexpr (VEC) {
        copy(g + (D - 1) * teams);
        mbar_wait(smem_u32(&full[team][slot]), parity, &aborted, a.status);
        if (++slot == D) slot = 0, parity ^= 1u;
      }
      if (n_mine <= 0) {
        if (VEC && lane == 0) mbar_arrive(read);
        continue;
      }
      const int past = a.V - g * kBeamGroup - lane * 8;  // logits from here on, for the lane
      const bool short_group = a.V - g * kBeamGroup < kBeamGroup;
      float2 x[N][kPer / 2];
      if constexpr (VEC) {
#pragma unroll
        for (int r = 0; r < N; ++r) staged(p + (N * pair + (r < n_mine ? r : 0)) * kBeamGroup, lane, x[r]);
        float2 y[kPer / 2];
        if (sh.base != nullptr) {
          staged(p + n_live * kBeamGroup, lane, y);
#pragma unroll
          for (int i = 0; i < kPer / 2; ++i)
#pragma unroll
            for (int r = 0; r < N; ++r) x[r][i] = add2(y[i], x[r][i]);
        }
        if (sh.prior != nullptr) {
          staged(reinterpret_cast<const float*>(p + (n_live + 1) * kBeamGroup), lane, y);
#pragma unroll
          for (int i = 0; i < kPer / 2; ++i) {
            y[i] = mul2(make_float2(sh.nbeta, sh.nbeta), y[i]);
#pragma unroll
            for (int r = 0; r < N; ++r) x[r][i] = add2(x[r][i], y[i]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(read);
        if (short_group) {
#pragma unroll
          for (int i = 0; i < kPer / 2; ++i)
            if (past <= (i >> 2) * 256) {
#pragma unroll
              for (int r = 0; r < N; ++r) x[r][i] = make_float2(neg_inf(), neg_inf());
            }
        }
      } else {
        load_single<T>(row, sh, g * kBeamGroup, a.V, lane, x);
      }
      float4 t[N];
      fold_group(x, lane, w, t);
#pragma unroll
      for (int r = 0; r < N; ++r)
        if (lane == r && r < n_mine) tops[r][g] = t[r];
    }
    __syncthreads();  // the block before has been joined, and all slots are read
#pragma unroll
    for (int r = 0; r < N; ++r) {
      float sum = r == 0 ? w.s.x + w.less.x : w.s.y + w.less.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, o);
      // (without a reference there is nothing to rescale: m = -inf and a sum of 0, or NaN)
      if (lane == r && r < n_mine)
        team_part[team][N * pair + r] =
            make_float2(w.m, w.limit[r] == neg_inf() || w.m == -w.nref[r] ? sum : sum * expf(-w.nref[r] - w.m));
    }
    __syncthreads();
    if (warp == 0 && lane < n_live) {
      float2 p = team_part[0][lane];
#pragma unroll 1
      for (int w = 1; w < teams; ++w) p = softmax_join(p, team_part[w][lane]);
      a.ws.part[(long long)(row0 + my_row) * a.parts + blockIdx.x - a.share.cta(block * a.groups)] = p;
    }
  }
  // copies that a wait gave up on land before the CTA exits
  if (VEC && *(volatile int*)&aborted != 0) {
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < kWaitLimitNs / 20) {
    }
  }
}

// ------------------------------------------------------------------ choosing the best of a list
namespace {

// The n-th largest of some keys, of which there are at least n, by bisection between their
// smallest lo and largest hi (of a lane); the bisection stops early at a value that n to
// `enough` keys reach.  count(mid): the lane's number of keys >= mid.
template <typename Count>
__device__ __forceinline__ uint32_t warp_kth(uint32_t lo, uint32_t hi, int n, int enough, Count count) {
  lo = __reduce_min_sync(kAllLanes, lo);
  hi = __reduce_max_sync(kAllLanes, hi);
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const int c = __reduce_add_sync(kAllLanes, count(mid));
    if (c >= n) {
      lo = mid;
      if (c <= enough) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// The n largest of the keys key(0..N-1) (n <= N), the lowest positions among equals:
// emit(slot, position, key) with ascending positions.
template <typename Key, typename Emit>
__device__ __forceinline__ void warp_top(int N, int n, Key key, Emit emit) {
  const int lane = threadIdx.x & 31;
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int i = lane; i < N; i += 32) {
    const uint32_t k = key(i);
    lo = min(lo, k);
    hi = max(hi, k);
  }
  const uint32_t T = warp_kth(lo, hi, n, n, [&](uint32_t mid) {
    int c = 0;
    for (int i = lane; i < N; i += 32) c += key(i) >= mid;
    return c;
  });
  int above = 0;
  for (int i = lane; i < N; i += 32) above += key(i) > T;
  int ties = n - __reduce_add_sync(kAllLanes, above), at = 0;
  for (int i0 = 0; i0 < N && at < n; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t k = i < N ? key(i) : 0u;
    const uint32_t before = (1u << lane) - 1u;
    const uint32_t same = __ballot_sync(kAllLanes, i < N && k == T);
    const bool tie = ((same >> lane) & 1u) && __popc(same & before) < ties;
    const uint32_t take = __ballot_sync(kAllLanes, (i < N && k > T) || tie);
    if ((take >> lane) & 1u) emit(at + __popc(take & before), i, k);
    at += __popc(take);
    ties -= min(ties, __popc(same));
  }
  __syncwarp();
}

__device__ __forceinline__ unsigned long long entry_key(uint32_t key, int token) {
  return ((unsigned long long)key << 32) | (unsigned long long)(0xFFFFFFFFu - (uint32_t)token);
}

// The finishing warp's own shared memory.
struct RowScratch {
  unsigned long long* list;  // [kBeamListCap] candidates
  int* quarters;             // [kBeamListCap] 4 group + quarter
  int* count;
};

// The row's `select` best logits by exact counting, however many are equal or crowd together
// in a few groups, into w.list.  The `select` best groups by (maximum, lowest group) hold
// them: a logit outside is beaten by one in each of those.
template <typename T>
__device__ __noinline__ void row_best_exact(const BeamSelectArgs& a, const T* logits, const Shared<T>& sh,
                                            const float4* tops, const RowScratch& w) {
  const int n_groups = min(a.select, a.groups);
  warp_top(a.groups, n_groups,
           [&](int i) {
             const float4 t = __ldcg(tops + i);
             return ordered_u32(fmax_nan(fmax3_nan(t.x, t.y, t.z), t.w));
           },
           [&](int slot, int i, uint32_t) { w.quarters[slot] = i; });
  // the groups ascend, so positions ascend with the tokens; only the last group can be short
  const int last = a.V - w.quarters[n_groups - 1] * kBeamGroup;
  const int total = (n_groups - 1) * kBeamGroup + min(kBeamGroup, last);
  auto token = [&](int p) { return w.quarters[p / kBeamGroup] * kBeamGroup + p % kBeamGroup; };
  warp_top(total, a.select, [&](int p) { return ordered_u32(mixed_logit<T>(logits, sh, token(p))); },
           [&](int slot, int p, uint32_t k) { w.list[slot] = entry_key(k, token(p)); });
}

// A bound that at least n of the maxima top[0..3] of all lanes reach (the n-th largest, or a
// little less: reading a few logits more takes less time than more bisection); 0 marks a
// missing one, and 0 is returned when fewer than n are there.
__device__ __forceinline__ uint32_t warp_bound(const uint32_t (&top)[4], int n) {
  uint32_t lo = 0xffffffffu, hi = 0;
  int some = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    lo = min(lo, top[r] == 0 ? 0xffffffffu : top[r]);
    hi = max(hi, top[r]);
    some += top[r] != 0;
  }
  if (__reduce_add_sync(kAllLanes, some) < n) return 0;
  return warp_kth(lo, hi, n, n + 2 + n / 4, [&](uint32_t mid) {
    return (top[0] >= mid) + (top[1] >= mid) + (top[2] >= mid) + (top[3] >= mid);
  });
}

// Four logits of a lane from a quarter; -inf past V.  The loads of the logits and of what they
// share leave together, before the first of them is used (volatile: in the order written), since
// each may take a microsecond to come.
template <typename T, bool VEC>
__device__ __forceinline__ void load_quarter(const BeamSelectArgs& a, const T* logits, const Shared<T>& sh, int quarter,
                                             int lane, float2 (&x)[2]) {
  const int v = (quarter >> 2) * kBeamGroup + quarter_offset<VEC>(quarter & 3, lane, 0);
  if constexpr (VEC) {
    const int u = v < a.V ? v : 0;
    Raw4<T> p, b;
    Raw4<float> pr;
    p.load(logits + u);
    if (sh.base != nullptr) b.load(sh.base + u);
    if (sh.prior != nullptr) pr.load(sh.prior + u);
    p.unpack(x);
    float2 y[2];
    if (sh.base != nullptr) {
      b.unpack(y);
      x[0] = add2(y[0], x[0]), x[1] = add2(y[1], x[1]);
    }
    if (sh.prior != nullptr) {
      const float2 nb = make_float2(sh.nbeta, sh.nbeta);
      pr.unpack(y);
      x[0] = add2(x[0], mul2(nb, y[0])), x[1] = add2(x[1], mul2(nb, y[1]));
    }
    if (v >= a.V) x[0] = x[1] = make_float2(neg_inf(), neg_inf());
  } else {
    x[0].x = v < a.V ? mixed_logit<T>(logits, sh, v) : neg_inf();
    x[0].y = v + 32 < a.V ? mixed_logit<T>(logits, sh, v + 32) : neg_inf();
    x[1].x = v + 64 < a.V ? mixed_logit<T>(logits, sh, v + 64) : neg_inf();
    x[1].y = v + 96 < a.V ? mixed_logit<T>(logits, sh, v + 96) : neg_inf();
  }
}

// take(x, quarter) for each listed quarter.
template <typename T, bool VEC, typename Take>
__device__ __forceinline__ void each_quarter(const BeamSelectArgs& a, const T* logits, const Shared<T>& sh,
                                             const int* quarters, int n_list, Take take) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int i = 0; i < n_list; i += 2) {  // two in flight
    float2 x[2], y[2];
    const int p = quarters[i], q = quarters[min(i + 1, n_list - 1)];
    load_quarter<T, VEC>(a, logits, sh, p, lane, x);
    load_quarter<T, VEC>(a, logits, sh, q, lane, y);
    take(x, p);
    if (i + 1 < n_list) take(y, q);
  }
}

// The row's `select` best logits or a few more, in any order, into w.list; returns their
// number.
template <typename T, bool VEC>
__device__ __forceinline__ int row_best(const BeamSelectArgs& a, const T* logits, const Shared<T>& sh,
                                        const float4* tops, const RowScratch& w) {
  const int lane = threadIdx.x & 31;
  const uint32_t none = ordered_u32(neg_inf());
  // A bound that `select` logits reach: from 128 maxima over the quarters of the groups
  // i, i + 32, ..., or, where there are hardly as many quarters as candidates (a small
  // vocabulary), over the logits themselves.
  const bool few = 4 * a.groups < 2 * a.select;
  uint32_t top[4] = {0, 0, 0, 0};
  if (!few) {
#pragma unroll 5
    for (int i = lane; i < a.groups; i += 32) {
      const float4 t = __ldcg(tops + i);
      top[0] = max(top[0], ordered_u32(t.x)), top[1] = max(top[1], ordered_u32(t.y));
      top[2] = max(top[2], ordered_u32(t.z)), top[3] = max(top[3], ordered_u32(t.w));
    }
  } else {
    for (int i = lane; i < 4 * a.groups; i += 32) w.quarters[i] = i;  // at most 2 select of them
    __syncwarp();
    each_quarter<T, VEC>(a, logits, sh, w.quarters, 4 * a.groups, [&](const float2(&x)[2], int) {
      top[0] = max(top[0], ordered_u32(x[0].x)), top[1] = max(top[1], ordered_u32(x[0].y));
      top[2] = max(top[2], ordered_u32(x[1].x)), top[3] = max(top[3], ordered_u32(x[1].y));
    });
  }
  uint32_t bound = warp_bound(top, a.select), rest = none;
  // With too little above -inf: all that is, and the lowest masked tokens.  Where more logits than
  // the list holds reach the bound, many of them mostly equal it (a mask of the type's lowest value,
  // constant rows): those above it, and the lowest tokens of the rest, 64 x 1 beams that take 16 with
  // one token allowed 65 us instead of 618.
  bool fill = bound <= none;
  if (fill) bound = none + 1;
#pragma unroll 1
  while (true) {
    const float floor = ordered_u32_to_float(bound);
    int n_list = 4 * a.groups;
    if (!few) {
      if (lane == 0) *w.count = 0;
      __syncwarp();
#pragma unroll 1
      for (int i = lane; i < a.groups; i += 32) {
        const float4 t = __ldcg(tops + i);
        // NaN counts as above every bound
        uint32_t reach =
            (t.x < floor ? 0u : 1u) | (t.y < floor ? 0u : 2u) | (t.z < floor ? 0u : 4u) | (t.w < floor ? 0u : 8u);
#pragma unroll 1
        for (; reach != 0; reach &= reach - 1) {
          const int slot = atomicAdd(w.count, 1);
          if (slot < kBeamListCap) w.quarters[slot] = 4 * i + __ffs((int)reach) - 1;
        }
      }
      __syncwarp();
      n_list = *w.count;
      __syncwarp();
    }
    if (lane == 0) *w.count = 0;
    __syncwarp();
    if (n_list <= kBeamListCap) {
      each_quarter<T, VEC>(a, logits, sh, w.quarters, n_list, [&](const float2(&x)[2], int q) {
        uint32_t reach = (x[0].x < floor ? 0u : 1u) | (x[0].y < floor ? 0u : 2u) | (x[1].x < floor ? 0u : 4u) |
                         (x[1].y < floor ? 0u : 8u);
#pragma unroll 1
        for (; reach != 0; reach &= reach - 1) {
          const int j = __ffs((int)reach) - 1;
          const float y = j & 2 ? (j & 1 ? x[1].y : x[1].x) : (j & 1 ? x[0].y : x[0].x);
          const int slot = atomicAdd(w.count, 1);
          const int token = (q >> 2) * kBeamGroup + quarter_offset<VEC>(q & 3, lane, j);
          if (slot < kBeamListCap) w.list[slot] = entry_key(ordered_u32(y), token);
        }
      });
      __syncwarp();
      int c = *w.count;
      __syncwarp();
      if (c <= kBeamListCap) {
        if (fill && c < a.select) {
          // at most c of the first select + c tokens are not masked; other values may be rarer
          const int end = rest == none ? a.V : min(a.V, kBeamFillTokens);
#pragma unroll 1
          for (int v0 = 0; v0 < end && c < a.select; v0 += 32) {
            const int v = v0 + lane;
            const bool equal = v < a.V && ordered_u32(mixed_logit<T>(logits, sh, v)) == rest;
            const uint32_t take = __ballot_sync(kAllLanes, equal);
            const int slot = c + __popc(take & ((1u << lane) - 1u));
            if (equal) w.list[slot] = entry_key(rest, v);  // slot < select + 32 <= kBeamListCap
            c += __popc(take);
          }
          __syncwarp();
        }
        if (c >= a.select) return c;
        break;
      }
    }
    if (fill || bound == 0xffffffffu) break;
    fill = true;
    rest = bound++;
  }
  row_best_exact<T>(a, logits, sh, tops, w);
  return a.select;
}

// Score of a logit in a row with (m, cum - log S) = st.
__device__ __forceinline__ float row_score(float x, float2 st) { return x == neg_inf() ? neg_inf() : (x - st.x) + st.y; }

// Group maxima of a lane at once, before the first of them is used: those of i, i + step, ...;
// -inf past the end (a maximum offered twice would raise the bound above too many others).
constexpr int kFinishLoads = 5;
__device__ __forceinline__ void load_tops(const float4* tops, int i, int step, int groups, float4 (&t)[kFinishLoads]) {
#pragma unroll
  for (int u = 0; u < kFinishLoads; ++u) t[u] = __ldcg(tops + min(i + u * step, groups - 1));
#pragma unroll
  for (int u = 1; u < kFinishLoads; ++u)
    if (i + u * step >= groups) t[u] = make_float4(neg_inf(), neg_inf(), neg_inf(), neg_inf());
}

// A candidate: (score, beam) and (x, token), both in the order in which larger is better.
struct Candidate {
  unsigned long long rank, within;
};

// The shared memory of a finishing CTA.
struct FinishScratch {
  float2* stat;      // [beams] maximum, cum - log S
  uint32_t* value;   // [values] scores of maxima
  Candidate* list;   // [kBeamFinishCap]
  int2* quarters;    // [kBeamFinishCap] (beam, 4 group + quarter)
  // for counting exactly: the beams' lists
  BeamEntry* entries;  // [beams * select]
  uint32_t* score;     // [beams * select]
  char* rows;          // a RowScratch for each warp
};

// The selection beam by beam: each one's `select` best candidates, then the best of those.
// However many scores are equal, masked, or crowd together.
template <typename T, bool VEC>
__device__ __noinline__ void finish_exact(const BeamSelectArgs& a, const FinishScratch& f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
  const int seq = blockIdx.x, n = a.select, total = a.beams * n;
  RowScratch w;
  w.list = reinterpret_cast<unsigned long long*>(f.rows) + warp * kBeamListCap;
  w.quarters = reinterpret_cast<int*>(f.rows + n_warps * kBeamListCap * 8) + warp * kBeamListCap;
  w.count = reinterpret_cast<int*>(f.rows + n_warps * kBeamListCap * 12) + warp;
  const Shared<T> sh = shared_terms<T>(a, seq);
#pragma unroll 1
  for (int k = warp; k < a.beams; k += n_warps) {
    const int row = seq * a.beams + k;
    BeamEntry* out = f.entries + k * n;
    const float2 st = f.stat[k];
    if (a.finished != nullptr && a.finished[row] != 0) {
      // one live candidate, the padding token; then the lowest other tokens at -inf
      for (int i = lane; i < n; i += 32) {
        out[i] = i == 0 ? BeamEntry{0.0f, a.pad_token} : BeamEntry{neg_inf(), i - 1 + (i - 1 >= a.pad_token)};
        f.score[k * n + i] = ordered_u32(row_score(out[i].x, st));
      }
      continue;
    }
    const int c = row_best<T, VEC>(a, static_cast<const T*>(a.logits) + (long long)row * a.ld, sh,
                                        a.ws.group_top + (long long)row * a.groups, w);
    __syncwarp();
    for (int i = lane; i < c; i += 32) {
      const unsigned long long mine = w.list[i];
      int rank = 0;
      for (int j = 0; j < c; ++j) rank += w.list[j] > mine;
      if (rank < n) {
        const float x = ordered_u32_to_float((uint32_t)(mine >> 32));
        out[rank] = BeamEntry{x, (int)(0xFFFFFFFFu - (uint32_t)mine)};
        f.score[k * n + rank] = ordered_u32(row_score(x, st));
      }
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp != 0) return;
  // (the warp's list is free again: at most kBeamMax positions and their keys)
  int* pos = w.quarters;
  uint32_t* pos_key = reinterpret_cast<uint32_t*>(w.list);
  warp_top(total, n, [&](int i) { return f.score[i]; },
           [&](int slot, int i, uint32_t k) { pos[slot] = i, pos_key[slot] = k; });
  for (int i = lane; i < n; i += 32) {
    // positions ascend with the slots, so equal scores keep the order of their slots
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += pos_key[j] > pos_key[i] || (pos_key[j] == pos_key[i] && j < i);
    const long long o = (long long)seq * n + rank;
    a.parents[o] = pos[i] / n;
    a.tokens[o] = f.entries[pos[i]].token;
    a.scores[o] = ordered_u32_to_float(pos_key[i]);
  }
}

}  // namespace

// A CTA per sequence; `finish_split` warps share a beam's groups.  The scores of group maxima,
// over all beams (of small vocabularies the logits'), bound the sequence's `select` best scores
// from below; few quarters reach the bound (about `select` of all beams together), and only
// they are read again, a warp each.
// Where the bound says little (masked rows, many equal scores, more candidates than the list
// holds) the CTA counts exactly, beam by beam.
//
// About 7 us for 64 x 8 or 1 x 4 beams of 151936 logits: a chain of dependent loads (maxima,
// bound, quarters), which more warps shorten.  A second CTA an SM would help many sequences
// less than the registers that it takes hurt (64 x 1 beams 1.5 us longer with 64 of them).
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kBeamFinishWarps, 1) beam_finish_kernel(BeamSelectArgs a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ int n_found, n_quarters;
  __shared__ uint32_t bound_key;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
  const int seq = blockIdx.x, n = a.select;
  const int split = a.finish_split;
  const int at_once = n_warps / split, part = warp % split;
  const int per_lane = a.finish_values;  // maxima a lane offers: 1 or 4
  const int values = a.beams * split * 32 * per_lane;
  FinishScratch f;
  f.stat = reinterpret_cast<float2*>(smem);
  char* rest = smem + (a.beams * 8 + 15) / 16 * 16;
  f.list = reinterpret_cast<Candidate*>(rest);
  f.quarters = reinterpret_cast<int2*>(f.list + kBeamFinishCap);
  f.value = reinterpret_cast<uint32_t*>(f.quarters + kBeamFinishCap);
  f.rows = rest;  // an exact count starts over, but for the rows' statistics
  f.entries = reinterpret_cast<BeamEntry*>(rest + n_warps * kBeamRowScratch);
  f.score = reinterpret_cast<uint32_t*>(f.entries + a.beams * n);
  if (threadIdx.x == 0) n_found = n_quarters = 0;
  const int run_blocks = (a.run_rows + a.scan_rows - 1) / a.scan_rows;
  pdl_wait();
  pdl_trigger();
#pragma unroll 1
  for (int k = warp / split; k < a.beams; k += at_once) {
    const int row = seq * a.beams + k;
    const bool done = a.finished != nullptr && a.finished[row] != 0;
    const float cum = __ldcg(a.cum + row);
    float2 st = make_float2(0.0f, cum);
    float top[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
    if (!done) {
      const int unit = (row / a.run_rows * run_blocks + row % a.run_rows / a.scan_rows) * a.groups;
      const int parts = a.share.cta(unit + a.groups - 1) - a.share.cta(unit) + 1;
      const float2* row_part = a.ws.part + (long long)row * a.parts;
      float2 p = __ldcg(row_part + min(lane, parts - 1));
      const float4* tops = a.ws.group_top + (long long)row * a.groups;
      if (a.finish_direct) {
        const Shared<T> sh = shared_terms<T>(a, seq);
        const T* logits = static_cast<const T*>(a.logits) + (long long)row * a.ld;
#pragma unroll 2
        for (int q = part; q < 4 * a.groups; q += split) {
          float2 x[2];
          load_quarter<T, VEC>(a, logits, sh, q, lane, x);
          top[0] = fmax_nan(top[0], x[0].x), top[1] = fmax_nan(top[1], x[0].y);
          top[2] = fmax_nan(top[2], x[1].x), top[3] = fmax_nan(top[3], x[1].y);
        }
      } else {
#pragma unroll 1
        for (int i = part * 32 + lane; i < a.groups; i += kFinishLoads * 32 * split) {
          float4 t[kFinishLoads];
          load_tops(tops, i, 32 * split, a.groups, t);
#pragma unroll
          for (int u = 0; u < kFinishLoads; ++u) {
            top[0] = fmax_nan(top[0], t[u].x), top[1] = fmax_nan(top[1], t[u].y);
            top[2] = fmax_nan(top[2], t[u].z), top[3] = fmax_nan(top[3], t[u].w);
          }
        }
      }
      if (lane >= parts) p = make_float2(neg_inf(), 0.0f);
#pragma unroll 1
      for (int i = lane + 32; i < parts; i += 32) p = softmax_join(p, __ldcg(row_part + i));
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) {
        const float2 q = make_float2(__shfl_down_sync(kAllLanes, p.x, o), __shfl_down_sync(kAllLanes, p.y, o));
        p = softmax_join(p, q);
      }
      st = make_float2(__shfl_sync(kAllLanes, p.x, 0), cum - logf(__shfl_sync(kAllLanes, p.y, 0)));
    } else if (part == 0 && lane == 0) {
      top[0] = 0.0f;  // the padding token
    }
    if (part == 0 && lane == 0) f.stat[k] = st;
    uint32_t* value = f.value + ((k * split + part) * 32 + lane) * per_lane;
    if (per_lane == 1) {
      value[0] = ordered_u32(row_score(fmax_nan(fmax3_nan(top[0], top[1], top[2]), top[3]), st));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) value[i] = ordered_u32(row_score(top[i], st));
    }
  }
  __syncthreads();
  if (warp == 0) {
    // up to 16 of the values of a lane in registers, so that the bisection hardly waits
    constexpr int R = 16;
    uint32_t v[R], lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool some = lane + 32 * i < values;
      v[i] = some ? f.value[lane + 32 * i] : 0u;
      lo = min(lo, some ? v[i] : 0xffffffffu);
      hi = max(hi, v[i]);
    }
    for (int i = lane + 32 * R; i < values; i += 32) {
      lo = min(lo, f.value[i]);
      hi = max(hi, f.value[i]);
    }
    const uint32_t key = warp_kth(lo, hi, n, n + 2 + n / 4, [&](uint32_t mid) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) c += v[i] >= mid;
      for (int i = lane + 32 * R; i < values; i += 32) c += f.value[i] >= mid;
      return c;
    });
    if (lane == 0) bound_key = key;
  }
  __syncthreads();
  const uint32_t none = ordered_u32(neg_inf());
  // With too little above -inf: all that is, and masked tokens for the rest.  (Above the largest
  // number there is NaN only, which says nothing of what else there is.)
  const bool fill = bound_key <= none, exact = bound_key == 0xffffffffu;
  const uint32_t key = fill ? none + 1 : bound_key;
  if (!exact) {
    const float bound = ordered_u32_to_float(key);
    auto found = [&](int k, float x, float score, int token) {
      const int slot = atomicAdd(&n_found, 1);
      if (slot < kBeamFinishCap)
        f.list[slot] = {((unsigned long long)ordered_u32(score) << 32) | (0xFFFFFFFFu - (uint32_t)k),
                        entry_key(ordered_u32(x), token)};
    };
#pragma unroll 1
    for (int k = warp / split; k < a.beams; k += at_once) {
      const int row = seq * a.beams + k;
      const float2 st = f.stat[k];
      if (a.finished != nullptr && a.finished[row] != 0) {
        if (part == 0 && lane == 0 && !(st.y < bound)) found(k, 0.0f, st.y, a.pad_token);
        continue;
      }
      // few lanes hold a maximum that reaches the bound
      const uint32_t* value = f.value + ((k * split + part) * 32 + lane) * per_lane;
      if (!a.finish_direct && value[0] < key &&
          (per_lane == 1 || max(max(value[1], value[2]), value[3]) < key))
        continue;
      const float4* tops = a.ws.group_top + (long long)row * a.groups;
#pragma unroll 1
      for (int i = part * 32 + lane; i < a.groups; i += kFinishLoads * 32 * split) {
        float4 t[kFinishLoads];
        load_tops(tops, i, 32 * split, a.groups, t);
#pragma unroll
        for (int u = 0; u < kFinishLoads; ++u) {
          const int g = i + u * 32 * split;
          // (a NaN reaches every bound)
          if (row_score(fmax_nan(fmax3_nan(t[u].x, t[u].y, t[u].z), t[u].w), st) < bound) continue;
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            if (row_score(q & 2 ? (q & 1 ? t[u].w : t[u].z) : (q & 1 ? t[u].y : t[u].x), st) < bound) continue;
            const int slot = atomicAdd(&n_quarters, 1);
            if (slot < kBeamFinishCap) f.quarters[slot] = make_int2(k, 4 * g + q);
          }
        }
      }
    }
    __syncthreads();
    const Shared<T> sh = shared_terms<T>(a, seq);
    const int n_list = min(n_quarters, kBeamFinishCap);
#pragma unroll 1
    for (int i = warp; i < n_list; i += n_warps) {
      const int k = f.quarters[i].x, q = f.quarters[i].y;
      const float2 st = f.stat[k];
      float2 x[2];
      load_quarter<T, VEC>(a, static_cast<const T*>(a.logits) + (long long)(seq * a.beams + k) * a.ld, sh, q, lane, x);
      if (row_score(fmax_nan(fmax3_nan(x[0].x, x[0].y, x[1].x), x[1].y), st) < bound) continue;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        const float y = j & 2 ? (j & 1 ? x[1].y : x[1].x) : (j & 1 ? x[0].y : x[0].x);
        const float score = row_score(y, st);
        if (!(score < bound)) found(k, y, score, (q >> 2) * kBeamGroup + quarter_offset<VEC>(q & 3, lane, j));
      }
    }
  }
  __syncthreads();
  int c = n_found;
  if (fill && c < n) {
    __syncthreads();  // all threads have taken this branch by the count that warp 0 now changes
    // The rest are masked tokens, the lowest of the lowest beam.  A beam whose own score is
    // not finite, or whose lowest logits fall out of fp32 below its maximum, has other candidates
    // at -inf, which an exact count sorts out.
    const int row = seq * a.beams;
    const bool done = a.finished != nullptr && a.finished[row] != 0;
    if (warp == 0 && row_score(-3.402823466e+38f, f.stat[0]) > neg_inf() && f.stat[0].y < -neg_inf()) {
      const Shared<T> sh = shared_terms<T>(a, seq);
      const T* logits = static_cast<const T*>(a.logits) + (long long)row * a.ld;
#pragma unroll 1
      for (int v0 = 0; v0 < a.V && c < n; v0 += 32) {
        const int v = v0 + lane;
        const bool masked = v < a.V && (done ? v != a.pad_token : mixed_logit<T>(logits, sh, v) == neg_inf());
        const uint32_t take = __ballot_sync(kAllLanes, masked);
        // at most select + 31 candidates
        if (masked) f.list[c + __popc(take & ((1u << lane) - 1u))] = {((unsigned long long)none << 32) | 0xFFFFFFFFu,
                                                                    entry_key(none, v)};
        c += __popc(take);
      }
      if (lane == 0) n_found = c;
    }
    __syncthreads();
    c = n_found;
  }
  if (exact || n_quarters > kBeamFinishCap || c < n || c > kBeamFinishCap) {
    finish_exact<T, VEC>(a, f);
    return;
  }
  for (int i = threadIdx.x; i < c; i += blockDim.x) {
    const Candidate mine = f.list[i];
    int rank = 0;
#pragma unroll 2
    for (int j = 0; j < c; ++j) {
      const Candidate other = f.list[j];
      rank += other.rank > mine.rank || (other.rank == mine.rank && other.within > mine.within);
    }
    if (rank < n) {
      const long long o = (long long)seq * n + rank;
      a.parents[o] = (int)(0xFFFFFFFFu - (uint32_t)mine.rank);
      a.tokens[o] = (long long)(0xFFFFFFFFu - (uint32_t)mine.within);
      a.scores[o] = ordered_u32_to_float((uint32_t)(mine.rank >> 32));
    }
  }
}

BeamKernel beam_scan_kernel_for(bool bf16, bool vec) {
  if (bf16) return vec ? beam_scan_kernel<__nv_bfloat16, true> : beam_scan_kernel<__nv_bfloat16, false>;
  return vec ? beam_scan_kernel<float, true> : beam_scan_kernel<float, false>;
}

BeamKernel beam_finish_kernel_for(bool bf16, bool vec) {
  if (bf16) return vec ? beam_finish_kernel<__nv_bfloat16, true> : beam_finish_kernel<__nv_bfloat16, false>;
  return vec ? beam_finish_kernel<float, true> : beam_finish_kernel<float, false>;
}

// --------------------------------------------------------------------------------
// Reordering.  dst[b, j] = src[b, parents[b, j]] for every state.  A tile is one piece of
// `chunk` bytes of all beams of one sequence: the rows that some child reads are staged in
// shared memory, then every child's piece is written from there, so each byte is read once
// however many children share a parent, and in place needs no second buffer.
//
// Bytes move 16 at a time whatever the alignment: a row is staged at its address modulo 16,
// and what is written to an aligned address is put together from five 32-bit words where
// source and destination differ modulo 16.
//
// Bound by memory: a cache of 8 beams in place, of which 597 MB have to be read and written for
// random parents (a row that keeps its place is neither), 98 us, 6.1 TB/s, 0.94 of a plain copy's
// rate; 64 x 8 GRU states of 2 KB and their histories 3.4 us, rows of 4099 bytes 3.8 us (13.3 when
// they moved by bytes), which is a launch and three passes of latency.
// --------------------------------------------------------------------------------
namespace {

// Starts the copy of `bytes` from src to stage + src % 16 (stage 16-byte aligned), by a warp
// that takes every `parts`-th run of 32 words.
__device__ __forceinline__ void stage_row(char* stage, const char* src, int bytes, int part, int parts, int lane) {
  const int shift = (int)(reinterpret_cast<uintptr_t>(src) & 15);
  char* dst = stage + shift;
  const int head = min(bytes, (16 - shift) & 15), words = (bytes - head) / 16, tail = bytes - head - 16 * words;
  const uint32_t d = smem_u32(dst + head);
  for (int i = part * 32 + lane; i < words; i += 32 * parts) cp_async_16(d + 16 * i, src + head + 16 * i, 16);
  if (part == 0) {
    if (lane < head) dst[lane] = src[lane];
    if (lane < tail) dst[bytes - tail + lane] = src[bytes - tail + lane];
  }
}

// Writes `bytes` from `from` in shared memory (any alignment) to dst, likewise.
__device__ __forceinline__ void write_row(char* dst, const char* from, int bytes, int part, int parts, int lane) {
  const int head = min(bytes, (int)(16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15);
  const int words = (bytes - head) / 16, tail = bytes - head - 16 * words;
  const char* p = from + head;
  uint4* out = reinterpret_cast<uint4*>(dst + head);
  const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);
  if (off == 0) {
    const uint4* in = reinterpret_cast<const uint4*>(p);
#pragma unroll 4
    for (int i = part * 32 + lane; i < words; i += 32 * parts) out[i] = in[i];
  } else {
    const uint32_t* in = reinterpret_cast<const uint32_t*>(p - (off & 3));
    const int bits = (off & 3) * 8;
#pragma unroll 2
    for (int i = part * 32 + lane; i < words; i += 32 * parts) {
      uint32_t w[5];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = in[4 * i + j];
      w[4] = bits != 0 ? in[4 * i + 4] : 0u;
      out[i] = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                          __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
    }
  }
  if (part == 0) {
    if (lane < head) dst[lane] = from[lane];
    if (lane < tail) dst[bytes - tail + lane] = from[bytes - tail + lane];
  }
}

}  // namespace

__global__ void __launch_bounds__(kBeamThreads)
    beam_reorder_kernel(const BeamReorderArgs a, const __grid_constant__ BeamStates states) {
  __shared__ __align__(16) char stage[kBeamReorderSmem];
  __shared__ int parent[kBeamMax];
  __shared__ unsigned long long used;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarps = kBeamThreads / 32;
  const int row_room = kBeamReorderSmem / a.beams & ~15;
  pdl_wait();
  pdl_trigger();
  for (long long tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    int k = 0;
    while (k + 1 < a.n_states && tile >= states.st[k + 1].tile0) ++k;
    const BeamState& st = states.st[k];
    const long long local = tile - st.tile0;
    const int c = (int)(local % st.chunks);
    const long long rest = local / st.chunks;
    const int o = (int)(rest % st.outer), seq = (int)(rest / st.outer);
    const bool in_place = st.src == st.dst;
    __syncthreads();  // the previous tile's stage and parents are no longer read
    if (threadIdx.x == 0) used = 0ull;
    __syncthreads();
    if (threadIdx.x < a.select) {
      int p = a.parents[(long long)seq * a.select + threadIdx.x];
      if (p < 0 || p >= a.beams) {
        // no such beam: the child keeps what it holds, and the status word says so
        if (a.status != nullptr) atomicCAS(a.status, 0, DELS_ERR_INVALID_ARG);
        p = -1;
      } else if (!(in_place && p == (int)threadIdx.x)) {
        atomicOr(&used, 1ull << p);
      }
      parent[threadIdx.x] = p;
    }
    __syncthreads();
    const long long at = (long long)c * st.chunk;
    const int bytes = (int)min((long long)st.chunk, st.inner - at);
    const char* src = st.src + (long long)seq * a.beams * st.src_row + o * st.src_outer + at;
    char* dst = st.dst + (long long)seq * a.select * st.dst_row + o * st.dst_outer + at;
    // a warp per row, or several where there are few
    const unsigned long long rows = used;
    int parts = a.beams < kWarps ? kWarps / a.beams : 1;
    for (int i = warp; i < a.beams * parts; i += kWarps) {
      const int r = i / parts;
      if ((rows >> r) & 1ull) stage_row(stage + r * row_room, src + r * st.src_row, bytes, i % parts, parts, lane);
    }
    cp_async_commit();
    cp_async_wait_all();
    __syncthreads();
    parts = a.select < kWarps ? kWarps / a.select : 1;
    for (int i = warp; i < a.select * parts; i += kWarps) {
      const int j = i / parts, p = parent[j];
      if (p < 0 || (in_place && p == j)) continue;
      const char* s = src + p * st.src_row;
      write_row(dst + j * st.dst_row, stage + p * row_room + (reinterpret_cast<uintptr_t>(s) & 15), bytes, i % parts,
                parts, lane);
    }
  }
}

}  // namespace dels
