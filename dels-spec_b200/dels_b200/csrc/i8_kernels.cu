// Rows to 8-bit integers:
//
//   a = max_k |x[k]|,  scale = a / 127,  q[k] = rint(x[k] * (127 / a))   (half to even)
//
// all in fp32.  A row of zeros has scale 0; a row with NaN or infinity has that scale and
// q = 0, so what is computed from it is NaN.
#include "i8_gemm.cuh"

namespace dels {

namespace {

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
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

}  // namespace

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const void* x, long long ld_x, int rows, int K,
                                                                      int8_t* q, long long ld_q, float* scale) {
  __shared__ float warp_top[kQuantThreads / 32];
  const int t = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* src = static_cast<const T*>(x) + (long long)row * ld_x;
    int8_t* dst = q + (long long)row * ld_q;
    const int whole = VEC ? K / 8 * 8 : 0;
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
    __syncthreads();
    if ((t & 31) == 0) warp_top[t >> 5] = top;
    __syncthreads();
    top = warp_top[0];
#pragma unroll
    for (int w = 1; w < kQuantThreads / 32; ++w) top = fmax_nan(top, warp_top[w]);
    // 127 / top overflows for a top below 2^-121: such rows are scaled up by a power of two
    // first, which changes no quotient
    const float up = top < 0x1p-100f ? 0x1p100f : 1.0f;
    const float inv = top > 0.0f && top <= 3.402823466e+38f ? __fdiv_rn(127.0f, top * up) : 0.0f;
    if (t == 0) scale[row] = __fdiv_rn(top, 127.0f);
    for (int k = t * 8; k < whole; k += kQuantThreads * 8) {
      float v[8];
      load8(src + k, v);
      uint32_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[h] = (uint32_t)(to_i8(v[4 * h] * up, inv) & 255) | (uint32_t)(to_i8(v[4 * h + 1] * up, inv) & 255) << 8 |
               (uint32_t)(to_i8(v[4 * h + 2] * up, inv) & 255) << 16 | (uint32_t)(to_i8(v[4 * h + 3] * up, inv) & 255) << 24;
      *reinterpret_cast<uint2*>(dst + k) = make_uint2(w[0], w[1]);
    }
    for (int k = whole + t; k < K; k += kQuantThreads) dst[k] = (int8_t)to_i8(to_f32(src[k]) * up, inv);
  }
}

QuantizeKernel quantize_rows_kernel_for(bool bf16, bool vec) {
  if (bf16) return vec ? quantize_rows_kernel<__nv_bfloat16, true> : quantize_rows_kernel<__nv_bfloat16, false>;
  return vec ? quantize_rows_kernel<float, true> : quantize_rows_kernel<float, false>;
}

}  // namespace dels
