// What the kernels of glp_linear share: the arguments, the activations, 16-bit packing.
#pragma once
#include "common.cuh"
#include "rowquant.cuh"

namespace glp {

enum Activation : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGeluTanh = 3, kActGeluErf = 4 };

struct LinearParams {
  int M, N, K;
  int dtype, out_dtype, activation;
  const void* x;
  const void* w;
  const void* w_up;
  int64_t ld_x, ld_w;
  const float* x_scale;
  const float* w_scale;
  const float* w_up_scale;
  const float* bias;
  const float* bias_up;
  const void* residual;
  void* y;
  int64_t ld_residual, ld_y;
  int* status;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// SiLU is v / (1 + e^-v) and tanh-GELU v / (1 + e^-2z), z = sqrt(2/pi) (v + 0.044715 v^3), which is
// 0.5 v (1 + tanh z) without its cancellation; both exponentials as 2^x with log2(e) folded into the
// constants.  Where the exponential overflows the quotient is -0, the limit.
__device__ __forceinline__ float act_relu(float v) { return v < 0.0f ? 0.0f : v; }  // a NaN stays
__device__ __forceinline__ float act_silu(float v) { return v * rcp_fast(1.0f + exp2_fast(-1.44269504f * v)); }
__device__ __forceinline__ float act_gelu_tanh(float v) {
  constexpr float c0 = -2.30220820f, c1 = -0.102943240f;  // -2 sqrt(2/pi) log2(e), and 0.044715 of it
  return v * rcp_fast(1.0f + exp2_fast(v * fmaf(c1 * v, v, c0)));
}
__device__ __forceinline__ float act_gelu_erf(float v) { return 0.5f * v * erfcf(-0.70710678f * v); }

__device__ __forceinline__ float activate(float v, int kind) {
  switch (kind) {
    case kActRelu: return act_relu(v);
    case kActSilu: return act_silu(v);
    case kActGeluTanh: return act_gelu_tanh(v);
    case kActGeluErf: return act_gelu_erf(v);
    default: return v;
  }
}

template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int kind) {
  if (kind == kActGeluTanh) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = act_gelu_tanh(v[j]);
  } else if (kind == kActSilu) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = act_silu(v[j]);
  } else if (kind == kActGeluErf) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = act_gelu_erf(v[j]);
  } else if (kind == kActRelu) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = act_relu(v[j]);
  }
}

// two outputs rounded to a 16-bit type (f16 beyond 65504 becomes an infinity), and back
__device__ __forceinline__ uint32_t pack16(float lo, float hi, int dtype) {
  if (dtype == kBF16) return pack_bf16(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void unpack16(uint32_t w, int dtype, float& lo, float& hi) {
  if (dtype == kBF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}

}  // namespace glp
