// y = act(x w^T xs ws + b) [* (x w_up^T xs wus + bu)] + residual for operands of any alignment:
// 64 x 64 output tiles, 256 threads of 4 x 4 outputs, 16 columns of K at a time through shared
// memory, one element per load.  Products are f32 FMAs (int8: exact int32 sums), which bound it: 32,768 x 768 x
// 1,153 bf16 with packed rows 3.7 ms (16 TFLOP/s), 96 us on the tensor cores with rows of 1,160; one row against
// 4,096 x 4,097 bf16, where 64 blocks walk K each by itself, 367 us, 11.1 us with rows of 4,104.
#pragma once
#include "linear.cuh"

namespace glp {

__device__ __forceinline__ float e4m3_to_f32(uint8_t c) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(c)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h2 & 0xffffu)));
}

template <int DT>
struct AnyAcc {
  using T = float;
};
template <>
struct AnyAcc<kI8> {
  using T = int;
};

template <int DT>
__device__ __forceinline__ typename AnyAcc<DT>::T load_operand(const void* p, int64_t i) {
  if constexpr (DT == kF16) return __half2float(static_cast<const __half*>(p)[i]);
  if constexpr (DT == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if constexpr (DT == kI8) return static_cast<const int8_t*>(p)[i];
  if constexpr (DT == kE4M3) return e4m3_to_f32(static_cast<const uint8_t*>(p)[i]);
}

template <int DT, bool GATED>
__global__ void __launch_bounds__(256) linear_any_kernel(const LinearParams p) {
  using T = typename AnyAcc<DT>::T;
  __shared__ T sx[16][65], sw[16][65], su[GATED ? 16 : 1][65];
  griddep_launch();
  griddep_wait();
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t n_tiles = (p.N + 63) / 64, tiles = n_tiles * ((p.M + 63) / 64);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t m0 = tile / n_tiles * 64, n0 = tile % n_tiles * 64;
    T acc[4][4] = {}, up[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 16 + ty, k = k0 + tx;
        const bool in_k = k < p.K;
        sx[tx][r] = in_k && m0 + r < p.M ? load_operand<DT>(p.x, (m0 + r) * p.ld_x + k) : T(0);
        sw[tx][r] = in_k && n0 + r < p.N ? load_operand<DT>(p.w, (n0 + r) * p.ld_w + k) : T(0);
        if constexpr (GATED) su[tx][r] = in_k && n0 + r < p.N ? load_operand<DT>(p.w_up, (n0 + r) * p.ld_w + k) : T(0);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        T a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = sx[k][ty + 16 * i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const T b = sw[k][tx + 16 * j];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i][j] += a[i] * b;
          if constexpr (GATED) {
            const T u = su[k][tx + 16 * j];
#pragma unroll
            for (int i = 0; i < 4; ++i) up[i][j] += a[i] * u;
          }
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + ty + 16 * i;
      if (m >= p.M) continue;
      const float xs = p.x_scale ? p.x_scale[m] : 1.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + tx + 16 * j;
        if (n >= p.N) continue;
        // (the sum first: the two scales' own product may leave f32's range where the value does not)
        float v = static_cast<float>(acc[i][j]) * xs;
        if (p.w_scale) v *= p.w_scale[n];
        if (p.bias) v += p.bias[n];
        float pair[2] = {v, v};
        activate_all(pair, p.activation);
        v = pair[0];
        if constexpr (GATED) {
          float u = static_cast<float>(up[i][j]) * xs;
          if (p.w_up_scale) u *= p.w_up_scale[n];
          if (p.bias_up) u += p.bias_up[n];
          v *= u;
        }
        if (p.residual) v += load_as_f32(p.residual, m * p.ld_residual + n, p.out_dtype);
        store_from_f32(p.y, m * p.ld_y + n, p.out_dtype, v);
      }
    }
  }
}

}  // namespace glp
