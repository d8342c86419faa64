// Rows to 8-bit integers, and their product with 8-bit weights for one or two rows.
//
//   a = max_k |x[k]|,  scale = a / 127,  q[k] = rint(x[k] * (127 / a))   (half to even)
//
// in fp32, every operation rounded by itself.  127 / a is one division for bf16 rows and
// 127 * (1 / a) for fp32 rows, as a tensor expression evaluates it: where x * 127 / a lies within
// a rounding of a half the two take neighbouring integers, and one integer of 200 000 moves an
// fp32 result by 5e-5, more than all its other roundings.  A row of zeros has scale 0; a row with
// NaN or infinity has that scale and q = 0, so what is computed from it is NaN.
//
// A block takes a row, reads it twice (the second time from L1 or L2) and writes it once.  512
// rows of 4096 bf16 take 3.9 us with 16-byte loads and 5.5 us where their alignment rules
// those out, 16 rows 2.6 and 4.8 us: latency at any size that a draft step has.
#include "i8_gemm.cuh"

namespace dels {

namespace {

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *(reinterpret_cast<const float4*>(p) + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  x[0] = bf16_lo(w.x), x[1] = bf16_hi(w.x), x[2] = bf16_lo(w.y), x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z), x[5] = bf16_hi(w.z), x[6] = bf16_lo(w.w), x[7] = bf16_hi(w.w);
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// |x * inv| <= 127 up to one rounding, so the clamp only catches that; a row that is not
// finite comes with inv = 0.
__device__ __forceinline__ int to_i8(float x, float inv) {
  const int v = inv == 0.0f ? 0 : __float2int_rn(__fmul_rn(x, inv));
  return max(-127, min(127, v));
}

// 8 values of a row as int8 (what 16-byte loads give), packed.
template <typename T>
__device__ __forceinline__ uint2 quantize8(const T* p, float up, float inv) {
  float v[8];
  load8(p, v);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = (uint32_t)(to_i8(v[4 * h] * up, inv) & 255) | (uint32_t)(to_i8(v[4 * h + 1] * up, inv) & 255) << 8 |
           (uint32_t)(to_i8(v[4 * h + 2] * up, inv) & 255) << 16 | (uint32_t)(to_i8(v[4 * h + 3] * up, inv) & 255) << 24;
  return make_uint2(w[0], w[1]);
}

// One row by the whole block (kQuantThreads threads); returns its scale.  warp_top: shared,
// a float for each warp.
template <typename T>
__device__ __forceinline__ float quantize_row(const T* src, int K, bool vec, int8_t* dst, float* warp_top) {
  const int t = threadIdx.x;
  const int whole = vec ? K / 8 * 8 : 0;
  float top = 0.0f;
  for (int k = t * 8; k < whole; k += kQuantThreads * 8) {
    float v[8];
    load8(src + k, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmax_nan(top, fabsf(v[j]));
  }
  for (int k = whole + t; k < K; k += kQuantThreads) top = fmax_nan(top, fabsf(to_f32(src[k])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  __syncthreads();  // warp_top of the row before has been read
  if ((t & 31) == 0) warp_top[t >> 5] = top;
  __syncthreads();
  top = warp_top[0];
#pragma unroll
  for (int w = 1; w < kQuantThreads / 32; ++w) top = fmax_nan(top, warp_top[w]);
  // 127 / top overflows for a top below 2^-121, 1 / top is denormal above 2^126: such rows are
  // scaled by a power of two first, which changes no quotient
  const float up = top < 0x1p-100f ? 0x1p100f : (top > 0x1p100f ? 0x1p-100f : 1.0f);
  float inv = 0.0f;
  if (top > 0.0f && top <= 3.402823466e+38f)
    inv = sizeof(T) == 2 ? __fdiv_rn(127.0f, top * up) : __fmul_rn(__frcp_rn(top * up), 127.0f);
  for (int k = t * 8; k < whole; k += kQuantThreads * 8) *reinterpret_cast<uint2*>(dst + k) = quantize8(src + k, up, inv);
  for (int k = whole + t; k < K; k += kQuantThreads) dst[k] = (int8_t)to_i8(to_f32(src[k]) * up, inv);
  return __fdiv_rn(top, 127.0f);
}

}  // namespace

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const void* x, long long ld_x, int rows, int K,
                                                                      int8_t* q, long long ld_q, float* scale) {
  __shared__ float warp_top[kQuantThreads / 32];
  pdl_wait();
  pdl_trigger();
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const float s = quantize_row(static_cast<const T*>(x) + (long long)row * ld_x, K, VEC, q + (long long)row * ld_q,
                                 warp_top);
    if (threadIdx.x == 0) scale[row] = s;
  }
}

QuantizeKernel quantize_rows_kernel_for(bool bf16, bool vec) {
  if (bf16) return vec ? quantize_rows_kernel<__nv_bfloat16, true> : quantize_rows_kernel<__nv_bfloat16, false>;
  return vec ? quantize_rows_kernel<float, true> : quantize_rows_kernel<float, false>;
}

// --------------------------------------------------------------------------------
// One or two rows: y[r, n] = (sum_k xq[r, k] w[n, k]) * sx[r] * sw[n] (+ bias[n]).
// Bound by the weights' bytes: 151936 channels of 4096 (622 MB) in 90 us for one row, 6.9 TB/s
// read, and by latency where they are few: 256 channels in 3.6 us.  A warp reads a channel with 16-byte loads, the next channel's
// first ones on their way while it adds up, and multiplies by dp4a; the sum is exact.
// --------------------------------------------------------------------------------
namespace {

__device__ __forceinline__ uint4 load_weights(const int8_t* p) {
  uint4 w;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
               : "l"(p));
  return w;
}

// ROWS: most rows; G: channels that a warp takes at a time, with kI8GemvLoads / G loads of a lane
// for each.  Dynamic shared memory: [ROWS][padded K] quantised rows, zero past K.
template <typename T, typename OutT, int ROWS, int G>
__global__ void __launch_bounds__(kI8GemvThreads, kI8GemvCtas) i8_gemv_kernel(I8GemvArgs a) {
  constexpr int kWarps = kI8GemvThreads / 32;
  constexpr int U = kI8GemvLoads, S = U / G;
  extern __shared__ __align__(16) int8_t rows_q[];
  __shared__ float warp_top[kWarps], scale[ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int padded = (a.K + 15) / 16 * 16, chunks = padded / 16, whole = a.K / 16;
  int n = (blockIdx.x * kWarps + warp) * G;
  uint4 w[U];
  // Chunks of 16 bytes of the channels from n0 on.  The last, partial one of a channel reaches
  // into the row's padding, whose products with the rows' zeros vanish; the last channel, with
  // no padding to rely on, adds its last bytes one by one.
  auto fetch = [&](int n0, int c0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int channel = n0 + u / S, c = c0 + u % S * 32 + lane;
      const int end = channel + 1 < a.n_out ? chunks : (channel < a.n_out ? whole : 0);
      w[u] = c < end ? load_weights(a.w + (long long)channel * a.ld_w + 16 * c) : make_uint4(0, 0, 0, 0);
    }
  };
  pdl_wait();  // (the kernel before this one may be the one that quantised the weights)
  pdl_trigger();
  fetch(n, 0);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    int8_t* dst = rows_q + r * padded;
    if (r >= a.rows) break;
    if constexpr (sizeof(T) == 1) {
      const int8_t* src = static_cast<const int8_t*>(a.x) + (long long)r * a.ld_x;
      for (int c = threadIdx.x; c < whole; c += kI8GemvThreads)
        reinterpret_cast<uint4*>(dst)[c] = reinterpret_cast<const uint4*>(src)[c];
      for (int k = 16 * whole + threadIdx.x; k < a.K; k += kI8GemvThreads) dst[k] = src[k];
      if (threadIdx.x == 0) scale[r] = a.sx[r];
    } else {
      const float s = quantize_row(static_cast<const T*>(a.x) + (long long)r * a.ld_x, a.K, a.vec != 0, dst, warp_top);
      if (threadIdx.x == 0) scale[r] = s;
    }
    for (int k = a.K + threadIdx.x; k < padded; k += kI8GemvThreads) dst[k] = 0;
  }
  __syncthreads();
  const int step = gridDim.x * kWarps * G;
#pragma unroll 1
  for (; n < a.n_out; n += step) {
    int acc[G][ROWS] = {};
    for (int c0 = 0; c0 < chunks; c0 += 32 * S) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = w[u];
      const bool more = c0 + 32 * S < chunks;
      fetch(more ? n : n + step, more ? c0 + 32 * S : 0);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int c = c0 + s * 32 + lane;
        if (c < chunks) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            if (r >= a.rows) break;
            const uint4 x = reinterpret_cast<const uint4*>(rows_q + r * padded)[c];
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const uint4 y = v[g * S + s];
              acc[g][r] = __dp4a((int)y.x, (int)x.x, acc[g][r]);
              acc[g][r] = __dp4a((int)y.y, (int)x.y, acc[g][r]);
              acc[g][r] = __dp4a((int)y.z, (int)x.z, acc[g][r]);
              acc[g][r] = __dp4a((int)y.w, (int)x.w, acc[g][r]);
            }
          }
        }
      }
    }
    if (n + G >= a.n_out && 16 * whole + lane < a.K) {
      const int k = 16 * whole + lane, byte = a.w[(long long)(a.n_out - 1) * a.ld_w + k];
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int g = 0; g < G; ++g)
          if (r < a.rows && n + g == a.n_out - 1) acc[g][r] += byte * rows_q[r * padded + k];
    }
    int mine = 0;  // lane G r + g: the sum of row r and channel g
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int total = __reduce_add_sync(0xffffffffu, acc[g][r]);
        mine = lane == G * r + g ? total : mine;
      }
    const int r = lane / G, channel = n + lane % G;
    if (r < a.rows && channel < a.n_out) {
      const float bias = a.bias != nullptr ? to_f32(static_cast<const OutT*>(a.bias)[channel]) : 0.0f;
      const float y = i8_result(mine, scale[r], a.sw[channel], bias);
      OutT* out = static_cast<OutT*>(a.out) + (long long)r * a.ld_out + channel;
      if constexpr (sizeof(OutT) == 2)
        *out = __float2bfloat16_rn(y);
      else
        *out = y;
    }
  }
}

template <typename T, typename OutT, int ROWS>
I8GemvKernel i8_gemv_channels(int channels) {
  if (channels == 4) return i8_gemv_kernel<T, OutT, ROWS, 4>;
  return channels == 2 ? i8_gemv_kernel<T, OutT, ROWS, 2> : i8_gemv_kernel<T, OutT, ROWS, 1>;
}

template <typename T, typename OutT>
I8GemvKernel i8_gemv_rows(int rows, int channels) {
  return rows <= 1 ? i8_gemv_channels<T, OutT, 1>(channels) : i8_gemv_channels<T, OutT, 2>(channels);
}

}  // namespace

I8GemvKernel i8_gemv_kernel_for(I8Source source, bool out_bf16, int rows, int channels) {
  switch (source) {
    case kI8FromInt8:
      return out_bf16 ? i8_gemv_rows<int8_t, __nv_bfloat16>(rows, channels) : i8_gemv_rows<int8_t, float>(rows, channels);
    case kI8FromBf16:
      return out_bf16 ? i8_gemv_rows<__nv_bfloat16, __nv_bfloat16>(rows, channels) : i8_gemv_rows<__nv_bfloat16, float>(rows, channels);
    default:
      return out_bf16 ? i8_gemv_rows<float, __nv_bfloat16>(rows, channels) : i8_gemv_rows<float, float>(rows, channels);
  }
}

}  // namespace dels
