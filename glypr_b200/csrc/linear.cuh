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

// The activations on two values at once (packed f32 pairs: half the FMA-pipe instructions).
//
// SiLU is v / (1 + e^-v) and tanh-GELU v / (1 + e^-2z), z = sqrt(2/pi) (v + 0.044715 v^3), which is
// 0.5 v (1 + tanh z) without its cancellation; both exponentials as 2^x with log2(e) folded into the
// constants.  Where the exponential overflows the quotient is -0, the limit.
//
// erf-GELU is max(v, 0) - 0.5 |v| erfc(|v| / sqrt 2).  With x = |v| / sqrt 2 and t = 1 / (1 + x/2),
// erfc(x) = t 2^(P(t - 0.6) - x^2 log2 e): log2(e^(x^2) erfc(x) / t) is smooth in t, and P is its
// minimax polynomial of degree 7 for x <= 11 (fitted for this file).  Relative error with f32 arithmetic: 1e-6 for
// |v| <= 1, and from there that of an exponent of up to 120 in f32: 3e-6 for |v| of 5 to 8, 8.4e-6 in the far
// tail.  |v| is cut at 64, where erfc is 0, so that an infinity stays one.
__device__ __forceinline__ float act_relu(float v) { return v < 0.0f ? 0.0f : v; }  // a NaN stays

__device__ __forceinline__ uint64_t act_sigmoid_like(uint64_t v, uint64_t x) {  // v / (1 + 2^x)
  float x0, x1, d0, d1;
  f2_split(x, x0, x1);
  f2_split(f2_add(f2(exp2_fast(x0), exp2_fast(x1)), f2(1.0f, 1.0f)), d0, d1);
  return f2_mul(v, f2(rcp_fast(d0), rcp_fast(d1)));
}
__device__ __forceinline__ uint64_t act_silu(uint64_t v) {
  return act_sigmoid_like(v, f2_mul(v, f2(-1.44269504f, -1.44269504f)));
}
__device__ __forceinline__ uint64_t act_gelu_tanh(uint64_t v) {
  constexpr float c0 = -2.30220820f, c1 = -0.102943240f;  // -2 sqrt(2/pi) log2(e), and 0.044715 of it
  return act_sigmoid_like(v, f2_mul(v, f2_fma(f2_mul(v, f2(c1, c1)), v, f2(c0, c0))));
}
__device__ __forceinline__ uint64_t act_gelu_erf(uint64_t v) {
  constexpr float c[8] = {-0.77293891f, 1.9785372f, 0.10157601f, -0.58963692f, -0.020841775f, 0.40999675f, -0.053513844f, -0.26732871f};
  float v0, v1, d0, d1, x0, x1;
  f2_split(v, v0, v1);
  const uint64_t a = f2(fminf(fabsf(v0), 64.0f), fminf(fabsf(v1), 64.0f));
  f2_split(f2_fma(a, f2(0.35355339f, 0.35355339f), f2(1.0f, 1.0f)), d0, d1);
  const uint64_t t = f2(rcp_fast(d0), rcp_fast(d1));
  const uint64_t s = f2_add(t, f2(-0.6f, -0.6f));
  uint64_t q = f2(c[7], c[7]);
#pragma unroll
  for (int i = 6; i >= 0; --i) q = f2_fma(q, s, f2(c[i], c[i]));
  f2_split(f2_fma(f2_mul(a, f2(-0.72134752f, -0.72134752f)), a, q), x0, x1);
  const uint64_t half = f2_mul(f2_mul(a, f2(-0.5f, -0.5f)), t);  // -0.5 |v| t
  return f2_fma(half, f2(exp2_fast(x0), exp2_fast(x1)), f2(act_relu(v0), act_relu(v1)));
}

template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int kind) {
  static_assert(N % 2 == 0, "pairs");
  if (kind == kActGeluTanh) {
#pragma unroll
    for (int j = 0; j < N; j += 2) f2_split(act_gelu_tanh(f2(v[j], v[j + 1])), v[j], v[j + 1]);
  } else if (kind == kActSilu) {
#pragma unroll
    for (int j = 0; j < N; j += 2) f2_split(act_silu(f2(v[j], v[j + 1])), v[j], v[j + 1]);
  } else if (kind == kActGeluErf) {
#pragma unroll
    for (int j = 0; j < N; j += 2) f2_split(act_gelu_erf(f2(v[j], v[j + 1])), v[j], v[j + 1]);
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
