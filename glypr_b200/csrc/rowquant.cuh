// Row kernels that write 8-bit rows with one f32 scale per row (int8 or e4m3 codes): the residual
// addition and RMS norm between two sublayers, and plain row quantisation.
//
//   x~ = x * rms(x) * post_gain   (or x),   h = (residual + x~) * layer_scalar,
//   n  = h * rms(h) * gain,   scale = max(max|n| / top, 2^-100),   code = rn(n / scale)
//
// Everything between the loads and the two roundings (h to its type, n to its code) is f32.
#pragma once
#include "common.cuh"

namespace glp {

enum DType : int { kF32 = 0, kF16 = 1, kBF16 = 2, kI8 = 3, kE4M3 = 4 };

constexpr float kQuantFloor = 7.8886090522101181e-31f;  // 2^-100
__host__ __device__ constexpr float quant_top(int q_dtype) { return q_dtype == kI8 ? 127.0f : 448.0f; }

struct RowQuantParams {
  int M, H;
  const void* x;
  const void* residual;
  const float* post_gain;
  const float* gain;
  void* h;
  void* q;
  float* scale;
  int64_t ld_x, ld_residual, ld_h, ld_q;
  float eps, layer_scalar;
  int x_dtype, h_dtype, q_dtype;
};

// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
  if (dtype == kF32) return static_cast<const float*>(p)[i];
  if (dtype == kF16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_from_f32(void* p, int64_t i, int dtype, float v) {
  if (dtype == kF32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == kF16)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// code of v (already divided by the scale), |v| <= top up to a few ulps.  int8: adding 1.5 * 2^23
// rounds to the nearest integer (ties to even) and leaves it in the low byte.
__device__ __forceinline__ uint8_t code_i8(float v) { return static_cast<uint8_t>(__float_as_uint(v + 12582912.0f)); }
__device__ __forceinline__ uint16_t code_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint8_t code_of(float v, int q_dtype) {
  return q_dtype == kI8 ? code_i8(v) : static_cast<uint8_t>(code_e4m3x2(v, 0.0f));
}

// sum of a and NaN-keeping maximum of b over the G threads that share a row (G a warp or the block)
template <int G>
__device__ __forceinline__ void row_reduce(float& a, float& b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
  }
  if constexpr (G > 32) {
    __shared__ float2 part[G / 32];
    const int w = threadIdx.x >> 5;
    __syncthreads();  // the previous reduction's readers are done
    if ((threadIdx.x & 31) == 0) part[w] = make_float2(a, b);
    __syncthreads();
    a = part[0].x, b = part[0].y;
#pragma unroll
    for (int i = 1; i < G / 32; ++i) {
      a += part[i].x;
      b = max_nan(b, part[i].y);
    }
  }
}

// the row's scale from its largest magnitude; NaN for one that is not finite, so that no code of the
// row (0 and -1 among them) stands for a number
__device__ __forceinline__ float scale_of(float amax, int q_dtype) {
  const float s = amax / quant_top(q_dtype);
  if (!(s < __int_as_float(0x7f800000))) return __int_as_float(0x7fffffff);
  return s < kQuantFloor ? kQuantFloor : s;
}

// One element at a time, any alignment: G threads per row, NC elements per thread, H <= G * NC.
// NORM false: plain row quantisation.
template <int G, int NC, bool NORM>
__global__ void __launch_bounds__(G < 128 ? 128 : G) row_quant_any_kernel(const RowQuantParams p) {
  constexpr int ROWS = G < 128 ? 128 / G : 1;
  const int t = threadIdx.x % G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / G;
  if (row >= p.M) return;  // whole warps or the whole block
  float v[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = c * G + t;
    v[c] = e < p.H ? load_as_f32(p.x, row * p.ld_x + e, p.x_dtype) : 0.0f;
  }
  float none = 0.0f;
  if constexpr (NORM) {
    float inv = 1.0f;
    if (p.post_gain) {
      float ss = 0.0f;
#pragma unroll
      for (int c = 0; c < NC; ++c) ss = fmaf(v[c], v[c], ss);
      row_reduce<G>(ss, none);
      inv = 1.0f / sqrtf(ss / static_cast<float>(p.H) + p.eps);
    }
    float ss = 0.0f, amax = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e = c * G + t;
      if (e < p.H) {
        float a = v[c];
        if (p.post_gain) a = a * inv * p.post_gain[e];
        if (p.residual) a += load_as_f32(p.residual, row * p.ld_residual + e, p.h_dtype);
        a *= p.layer_scalar;
        if (p.h) store_from_f32(p.h, row * p.ld_h + e, p.h_dtype, a);
        ss = fmaf(a, a, ss);
        v[c] = p.gain ? a * p.gain[e] : a;
        amax = max_nan(amax, fabsf(v[c]));
      }
    }
    row_reduce<G>(ss, amax);
    const float inv_h = 1.0f / sqrtf(ss / static_cast<float>(p.H) + p.eps);
    const float s = scale_of(amax * inv_h, p.q_dtype);
    const float k = inv_h / s;
    if (t == 0) p.scale[row] = s;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e = c * G + t;
      if (e < p.H) static_cast<uint8_t*>(p.q)[row * p.ld_q + e] = code_of(v[c] * k, p.q_dtype);
    }
  } else {
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) amax = max_nan(amax, fabsf(v[c]));
    row_reduce<G>(none, amax);
    const float s = scale_of(amax, p.q_dtype);
    const float k = 1.0f / s;
    if (t == 0) p.scale[row] = s;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e = c * G + t;
      if (e < p.H) static_cast<uint8_t*>(p.q)[row * p.ld_q + e] = code_of(v[c] * k, p.q_dtype);
    }
  }
}

}  // namespace glp
