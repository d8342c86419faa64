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
//   beam_scan_kernel   one pass over the logits: per slice of a row the running (m, S) of
//                      an online softmax, and the maximum of every group of logits.
//   beam_row_kernel    the row's `select` best groups by (maximum, lowest group) hold its
//                      `select` best logits: a logit outside them is beaten by one in each.
//                      They are read again and their best logits kept, in order.
//   beam_merge_kernel  scores of all beams' lists, the best `select` of them.
#include "beam_kernels.cuh"

namespace dels {

namespace {

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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// (m, s) of two parts of a softmax; s counts exp(x - m).
__device__ __forceinline__ float2 softmax_join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  // a part without any finite logit has s = 0 (or NaN) and may have m = -inf
  const float ea = a.x == m ? 1.0f : __expf(a.x - m);
  const float eb = b.x == m ? 1.0f : __expf(b.x - m);
  return make_float2(m, a.y * ea + b.y * eb);
}

// x[v] of one logit.  Every operation is rounded by itself, in this order.
template <typename T, bool MIX>
__device__ __forceinline__ float mixed_logit(const T* row, const T* base, const float* prior, float beta, int v) {
  float x = to_f32(row[v]);
  if constexpr (MIX) {
    if (base != nullptr) x = __fadd_rn(to_f32(base[v]), x);
    if (prior != nullptr) x = __fsub_rn(x, __fmul_rn(beta, __ldg(prior + v)));
  }
  return x;
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
  const float4 b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p));
  x[0] = bf16_lo(w.x), x[1] = bf16_hi(w.x), x[2] = bf16_lo(w.y), x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z), x[5] = bf16_hi(w.z), x[6] = bf16_lo(w.w), x[7] = bf16_hi(w.w);
}

// Positions of the n largest of keys[0..N) in shared memory (equal keys: lowest positions),
// ascending, into pos[0..n).  All threads of the block call it; n <= N, n <= kBeamMax.
// The n-th largest key comes from a bisection over the keys' common leading bits; then one
// warp walks the keys in order.
__device__ void block_top_positions(const uint32_t* keys, int N, int n, int* pos, uint32_t* shared4) {
  const int t = threadIdx.x;
  if (N <= n) {
    for (int i = t; i < N; i += kBeamThreads) pos[i] = i;
    __syncthreads();
    return;
  }
  // shared4[0]: count of the bisection step, [1] / [2]: smallest and largest key
  if (t == 0) shared4[0] = 0, shared4[1] = 0xFFFFFFFFu, shared4[2] = 0;
  __syncthreads();
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  for (int i = t; i < N; i += kBeamThreads) {
    lo = min(lo, keys[i]);
    hi = max(hi, keys[i]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if ((t & 31) == 0) {
    atomicMin(&shared4[1], lo);
    atomicMax(&shared4[2], hi);
  }
  __syncthreads();
  lo = shared4[1];
  hi = shared4[2];
  // largest T with count(keys >= T) >= n, in [lo, hi]
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    int c = 0;
    for (int i = t; i < N; i += kBeamThreads) c += keys[i] >= mid;
    c = __reduce_add_sync(0xffffffffu, c);
    if ((t & 31) == 0) atomicAdd(&shared4[0], (uint32_t)c);
    __syncthreads();
    const uint32_t total = shared4[0];
    __syncthreads();
    if (t == 0) shared4[0] = 0;
    __syncthreads();
    if (total >= (uint32_t)n) {
      lo = mid;
      if (total == (uint32_t)n) break;
    } else {
      hi = mid - 1;
    }
  }
  if (t < 32) {
    int above = 0;
    for (int i = t; i < N; i += 32) above += keys[i] > lo;
    above = __reduce_add_sync(0xffffffffu, above);
    // above < n unless the bisection stopped early on an exact count, when it is <= n
    int ties = n - above, at = 0;
    for (int i0 = 0; i0 < N && at < n; i0 += 32) {
      const int i = i0 + t;
      const uint32_t k = i < N ? keys[i] : 0u;
      const uint32_t same = __ballot_sync(0xffffffffu, i < N && k == lo);
      const bool tie = i < N && k == lo && __popc(same & ((1u << t) - 1u)) < ties;
      const uint32_t take = __ballot_sync(0xffffffffu, (i < N && k > lo) || tie);
      if ((take >> t) & 1u) pos[at + __popc(take & ((1u << t) - 1u))] = i;
      at += __popc(take);
      ties -= min(ties, __popc(same));
    }
  }
  __syncthreads();
}

}  // namespace

template <typename T, bool MIX, bool VEC>
__global__ void __launch_bounds__(kBeamThreads) beam_scan_kernel(const BeamSelectArgs a) {
  __shared__ float2 warp_part[kBeamThreads / 32];
  const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  if (a.finished != nullptr && a.finished[row] != 0) return;
  const T* logits = static_cast<const T*>(a.logits) + (long long)row * a.ld;
  const T* base = nullptr;
  float beta = 0.0f;
  if constexpr (MIX) {
    if (a.base != nullptr) base = static_cast<const T*>(a.base) + (long long)(row / a.beams) * a.ld_base;
    if (a.prior != nullptr) beta = __ldg(a.beta);
  }
  const int per_slice = (a.groups + a.slices - 1) / a.slices;
  const int g_end = min(a.groups, (slice + 1) * per_slice);
  float m = neg_inf(), s = 0.0f;  // m is the same in all lanes, s the lane's own sum
  for (int g = slice * per_slice + warp; g < g_end; g += kBeamThreads / 32) {
    const int v0 = g * kBeamGroup;
    float x[8];
    if (VEC && v0 + kBeamGroup <= a.V) {
      const int v = v0 + lane * 8;
      load8(logits + v, x);
      if constexpr (MIX) {
        if (base != nullptr) {
          float b[8];
          load8(base + v, b);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = __fadd_rn(b[j], x[j]);
        }
        if (a.prior != nullptr) {
          const float4 p = __ldg(reinterpret_cast<const float4*>(a.prior + v));
          const float4 q = __ldg(reinterpret_cast<const float4*>(a.prior + v) + 1);
          const float pr[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = __fsub_rn(x[j], __fmul_rn(beta, pr[j]));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int v = v0 + j * 32 + lane;
        x[j] = v < a.V ? mixed_logit<T, MIX>(logits, base, a.prior, beta, v) : neg_inf();
      }
    }
    float top = fmax_nan(fmax3_nan(x[0], x[1], x[2]), fmax3_nan(x[3], x[4], x[5]));
    top = warp_max_nan(fmax3_nan(top, x[6], x[7]));
    if (top > m) {
      s *= __expf(m - top);  // m = -inf: s is 0 and stays 0
      m = top;
    }
    const float ref = m == neg_inf() ? 0.0f : m;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += __expf(x[j] - ref);
    if (lane == 0) a.ws.group_key[(long long)row * a.groups + g] = ordered_u32(top);
  }
  s = warp_sum(s);
  if (lane == 0) warp_part[warp] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x == 0) {
    float2 p = warp_part[0];
    for (int w = 1; w < kBeamThreads / 32; ++w) p = softmax_join(p, warp_part[w]);
    a.ws.part[(long long)row * a.slices + slice] = p;
  }
}

// Dynamic shared memory: keys [max(groups, select * kBeamGroup)] uint32.
template <typename T, bool MIX>
__global__ void __launch_bounds__(kBeamThreads) beam_row_kernel(const BeamSelectArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t shared4[4];
  __shared__ int groups[kBeamMax], pos[kBeamMax];
  __shared__ unsigned long long best[kBeamMax];
  const int row = blockIdx.x, t = threadIdx.x;
  pdl_wait();
  BeamEntry* out = a.ws.best + (long long)row * a.select;
  if (a.finished != nullptr && a.finished[row] != 0) {
    // one live candidate, the padding token; then the lowest other tokens at -inf
    for (int i = t; i < a.select; i += kBeamThreads) {
      const int rest = i - 1 + (i - 1 >= a.pad_token);
      out[i] = i == 0 ? BeamEntry{0.0f, a.pad_token} : BeamEntry{neg_inf(), rest};
    }
    if (t == 0) a.ws.stat[row] = make_float2(0.0f, a.cum[row]);
    return;
  }
  if (t == 0) {
    const float2* part = a.ws.part + (long long)row * a.slices;
    float2 p = part[0];
    for (int i = 1; i < a.slices; ++i) p = softmax_join(p, part[i]);
    a.ws.stat[row] = make_float2(p.x, a.cum[row] - logf(p.y));
  }
  for (int g = t; g < a.groups; g += kBeamThreads) keys[g] = a.ws.group_key[(long long)row * a.groups + g];
  __syncthreads();
  const int n_groups = min(a.select, a.groups);
  block_top_positions(keys, a.groups, n_groups, groups, shared4);
  const T* logits = static_cast<const T*>(a.logits) + (long long)row * a.ld;
  const T* base = nullptr;
  float beta = 0.0f;
  if constexpr (MIX) {
    if (a.base != nullptr) base = static_cast<const T*>(a.base) + (long long)(row / a.beams) * a.ld_base;
    if (a.prior != nullptr) beta = __ldg(a.beta);
  }
  // the groups ascend, so positions ascend with the tokens; only the last group can be
  // short, and it is the last one here
  int total = 0;
  for (int i = 0; i < n_groups; ++i) {
    const int v0 = groups[i] * kBeamGroup, len = min(kBeamGroup, a.V - v0);
    for (int j = t; j < len; j += kBeamThreads)
      keys[total + j] = ordered_u32(mixed_logit<T, MIX>(logits, base, a.prior, beta, v0 + j));
    total += len;
  }
  __syncthreads();
  block_top_positions(keys, total, a.select, pos, shared4);
  if (t < a.select) {
    const int p = pos[t];
    const int token = groups[p / kBeamGroup] * kBeamGroup + p % kBeamGroup;
    best[t] = ((unsigned long long)keys[p] << 32) | (unsigned long long)(0xFFFFFFFFu - (uint32_t)token);
  }
  __syncthreads();
  if (t < a.select) {
    int rank = 0;
    for (int i = 0; i < a.select; ++i) rank += best[i] > best[t];
    out[rank] = BeamEntry{ordered_u32_to_float((uint32_t)(best[t] >> 32)),
                          (int)(0xFFFFFFFFu - (uint32_t)(best[t] & 0xFFFFFFFFull))};
  }
}

// Dynamic shared memory: keys [beams * select] uint32.
__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const BeamSelectArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t shared4[4];
  __shared__ int pos[kBeamMax];
  __shared__ unsigned long long best[kBeamMax];
  const int seq = blockIdx.x, t = threadIdx.x;
  pdl_wait();
  const BeamEntry* lists = a.ws.best + (long long)seq * a.beams * a.select;
  const int total = a.beams * a.select;
  for (int i = t; i < total; i += kBeamThreads) {
    const float2 st = a.ws.stat[seq * a.beams + i / a.select];
    const float x = lists[i].x;
    keys[i] = ordered_u32(x == neg_inf() ? neg_inf() : (x - st.x) + st.y);
  }
  __syncthreads();
  block_top_positions(keys, total, a.select, pos, shared4);
  if (t < a.select)
    best[t] = ((unsigned long long)keys[pos[t]] << 32) | (unsigned long long)(0xFFFFFFFFu - (uint32_t)pos[t]);
  __syncthreads();
  if (t < a.select) {
    int rank = 0;
    for (int i = 0; i < a.select; ++i) rank += best[i] > best[t];
    const long long o = (long long)seq * a.select + rank;
    a.parents[o] = pos[t] / a.select;
    a.tokens[o] = lists[pos[t]].token;
    a.scores[o] = ordered_u32_to_float(keys[pos[t]]);
  }
}

template __global__ void beam_scan_kernel<float, false, false>(const BeamSelectArgs);
template __global__ void beam_scan_kernel<float, false, true>(const BeamSelectArgs);
template __global__ void beam_scan_kernel<float, true, false>(const BeamSelectArgs);
template __global__ void beam_scan_kernel<float, true, true>(const BeamSelectArgs);
template __global__ void beam_scan_kernel<__nv_bfloat16, false, false>(const BeamSelectArgs);
template __global__ void beam_scan_kernel<__nv_bfloat16, false, true>(const BeamSelectArgs);
template __global__ void beam_scan_kernel<__nv_bfloat16, true, false>(const BeamSelectArgs);
template __global__ void beam_scan_kernel<__nv_bfloat16, true, true>(const BeamSelectArgs);
template __global__ void beam_row_kernel<float, false>(const BeamSelectArgs);
template __global__ void beam_row_kernel<float, true>(const BeamSelectArgs);
template __global__ void beam_row_kernel<__nv_bfloat16, false>(const BeamSelectArgs);
template __global__ void beam_row_kernel<__nv_bfloat16, true>(const BeamSelectArgs);

// --------------------------------------------------------------------------------
// Reordering.  dst[b, j] = src[b, parents[b, j]] for every state.  A tile is one piece of
// `chunk` bytes of all beams of one sequence: the rows that some child reads are staged in
// shared memory, then every child's piece is written from there, so each byte is read once
// however many children share a parent, and in place needs no second buffer.
// --------------------------------------------------------------------------------
namespace {

template <typename W>
__device__ __forceinline__ void reorder_tile(const BeamState& st, const char* src, char* dst, int bytes, int beams,
                                             int select, unsigned long long used, const int* parent, bool in_place,
                                             char* stage) {
  const int words = bytes / (int)sizeof(W);
  for (int r = 0; r < beams; ++r) {
    if (!((used >> r) & 1ull)) continue;
    const W* s = reinterpret_cast<const W*>(src + r * st.src_row);
    W* d = reinterpret_cast<W*>(stage + r * st.chunk);
    for (int i = threadIdx.x; i < words; i += blockDim.x) d[i] = s[i];
  }
  __syncthreads();
  for (int j = 0; j < select; ++j) {
    const int p = parent[j];
    if (p < 0 || (in_place && p == j)) continue;
    const W* s = reinterpret_cast<const W*>(stage + p * st.chunk);
    W* d = reinterpret_cast<W*>(dst + j * st.dst_row);
    for (int i = threadIdx.x; i < words; i += blockDim.x) d[i] = s[i];
  }
}

}  // namespace

__global__ void __launch_bounds__(kBeamThreads) beam_reorder_kernel(const __grid_constant__ BeamReorderArgs a) {
  __shared__ __align__(16) char stage[kBeamReorderSmem];
  __shared__ int parent[kBeamMax];
  __shared__ unsigned long long used;
  pdl_wait();
  for (long long tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    int k = 0;
    while (k + 1 < a.n_states && tile >= a.st[k + 1].tile0) ++k;
    const BeamState& st = a.st[k];
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
    switch (st.width) {
      case 16: reorder_tile<uint4>(st, src, dst, bytes, a.beams, a.select, used, parent, in_place, stage); break;
      case 8: reorder_tile<uint2>(st, src, dst, bytes, a.beams, a.select, used, parent, in_place, stage); break;
      case 4: reorder_tile<uint32_t>(st, src, dst, bytes, a.beams, a.select, used, parent, in_place, stage); break;
      case 2: reorder_tile<uint16_t>(st, src, dst, bytes, a.beams, a.select, used, parent, in_place, stage); break;
      default: reorder_tile<uint8_t>(st, src, dst, bytes, a.beams, a.select, used, parent, in_place, stage); break;
    }
  }
}

}  // namespace dels
