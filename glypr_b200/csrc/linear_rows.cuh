// glp_linear for few rows of x (single tokens, short batches): the time is the weights' way from memory,
// so every warp of the device reads a piece of them with 16-byte loads straight into the fragments of
// mma.sync, without shared memory in between.
//
// One MMA multiplies 16 rows of x by 8 rows of w.  A fragment register holds neighbouring elements of K,
// and which elements those are does not matter as long as x and w agree: lane (g, t) takes the 16 bytes
// at K offset 64 s + 16 t of row g of w and of rows g and g + 8 of x, which are the fragments of two
// MMAs.  Four lanes read 64 contiguous bytes of a row.  A block owns 8 R rows of w (and the same of
// w_up), its warps take the 64-byte steps of K in turn, and their sums are added in warp order, so a
// result does not depend on timing.
//
// Many short-lived warps beat few with long prefetch queues: with 16 warps a block and two steps in flight each,
// one row against 4,096 x 4,096 f16 weights takes 6.1 us where they stay in L2 and 9.5 us from memory (4 warps with
// 8 steps ahead: 12.9 us), gated 2 x 1,152 x 768 bf16 2.6 and 3.0 us, 3 x 8,191 x 4,096 e4m3 9.2 and 11.3 us, in a
// CUDA graph and so without the host's launch time.  From memory the large ones read at 3.0 to 3.5 TB/s, about half
// of the copy rate: what bounds them is latency, for each block drains its loads before its warps' sums are
// joined, and there are more blocks than fit at once.  Past 32 rows x itself, read again by every block, is the
// larger stream.
#pragma once
#include "common.cuh"
#include "linear.cuh"

namespace glp {

template <int DT>
struct RowsAcc {
  using T = float;
};
template <>
struct RowsAcc<kI8> {
  using T = int;
};

// d += a (16 x 32 bytes of x) * b (8 x 32 bytes of w)^T
template <int DT>
__device__ __forceinline__ void mma_rows(typename RowsAcc<DT>::T (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
#define GLP_MMA(shape, types, c)                                                                              \
  asm volatile("mma.sync.aligned." shape ".row.col." types " {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" \
               : c(d[0]), c(d[1]), c(d[2]), c(d[3])                                                           \
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
  if constexpr (DT == kF16) GLP_MMA("m16n8k16", "f32.f16.f16.f32", "+f");
  if constexpr (DT == kBF16) GLP_MMA("m16n8k16", "f32.bf16.bf16.f32", "+f");
  if constexpr (DT == kE4M3) GLP_MMA("m16n8k32", "f32.e4m3.e4m3.f32", "+f");
  if constexpr (DT == kI8) GLP_MMA("m16n8k32", "s32.s8.s8.s32", "+r");
#undef GLP_MMA
}

// 16 bytes at byte offset b of a row of `bytes` bytes, zeros past its end.  Coherent loads: under a dependent
// launch this kernel is already resident while the one before it writes x (or w), so neither is read-only
// for the kernel's life, which the non-coherent path asks for; volatile, so that none moves over the wait.
template <bool STREAM>
__device__ __forceinline__ uint4 load16(const uint8_t* row, int b, int bytes) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (b + 16 <= bytes) {
    if constexpr (STREAM)
      v = ld_stream(row + b);
    else
      asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                   : "l"(row + b));
  } else if (b < bytes) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (b + i < bytes) w[i / 4] |= static_cast<uint32_t>(row[b + i]) << (8 * (i & 3));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}

// M <= 16 MT; a block of WARPS warps owns 8 R rows of w; U steps of K in flight per warp
template <int DT, bool GATED, int MT, int R, int U, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) linear_rows_kernel(const LinearParams p) {
  using T = typename RowsAcc<DT>::T;
  constexpr int ES = DT == kF16 || DT == kBF16 ? 2 : 1;
  constexpr int NW = GATED ? 2 : 1;
  constexpr int COLS = 8 * R, OUTS = MT * 16 * COLS;  // outputs of the block
  constexpr int THREADS = 32 * WARPS, PER = (OUTS + THREADS - 1) / THREADS;  // ... per thread
  __shared__ T part[WARPS][NW][OUTS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * COLS;
  const int bytes = p.K * ES, steps = (bytes + 63) / 64;
  griddep_launch();
  griddep_wait();
  // what the epilogue needs besides the sums, on its way during the products
  float xs[PER], ws[PER], wus[PER], b[PER], bu[PER], res[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int o = threadIdx.x + THREADS * i;
    const int64_t m = o / COLS, n = n0 + o % COLS;
    const bool in = m < p.M && n < p.N;
    xs[i] = in && p.x_scale ? p.x_scale[m] : 1.0f;
    ws[i] = in && p.w_scale ? p.w_scale[n] : 1.0f;
    b[i] = in && p.bias ? p.bias[n] : 0.0f;
    wus[i] = GATED && in && p.w_up_scale ? p.w_up_scale[n] : 1.0f;
    bu[i] = GATED && in && p.bias_up ? p.bias_up[n] : 0.0f;
    res[i] = in && p.residual ? load_as_f32(p.residual, m * p.ld_residual + n, p.out_dtype) : 0.0f;
  }
  const uint8_t* wr = static_cast<const uint8_t*>(p.w) + (n0 + g) * p.ld_w * ES;
  const uint8_t* ur = static_cast<const uint8_t*>(p.w_up) + (n0 + g) * p.ld_w * ES;
  const int64_t w_step = 8 * p.ld_w * ES;
  const uint8_t* xr = static_cast<const uint8_t*>(p.x);
  T acc[NW][R][MT][4];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[w][r][mt][i] = T(0);
  for (int s0 = warp; s0 < steps; s0 += WARPS * U) {
    uint4 wv[NW][R][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = (s0 + WARPS * u) * 64 + t * 16;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int wbytes = n0 + 8 * r + g < p.N ? bytes : 0;  // a row past N reads as zeros
        wv[0][r][u] = load16<true>(wr + r * w_step, at, wbytes);
        if constexpr (GATED) wv[1][r][u] = load16<true>(ur + r * w_step, at, wbytes);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = (s0 + WARPS * u) * 64 + t * 16;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int m = mt * 16 + g;
        const uint4 lo = load16<false>(xr + m * p.ld_x * ES, at, m < p.M ? bytes : 0);
        const uint4 hi = load16<false>(xr + (m + 8) * p.ld_x * ES, at, m + 8 < p.M ? bytes : 0);
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            mma_rows<DT>(acc[w][r][mt], lo.x, hi.x, lo.y, hi.y, wv[w][r][u].x, wv[w][r][u].y);
            mma_rows<DT>(acc[w][r][mt], lo.z, hi.z, lo.w, hi.w, wv[w][r][u].z, wv[w][r][u].w);
          }
      }
    }
  }
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i)  // lane (g, t) holds rows g, g + 8 and columns 2 t, 2 t + 1
          part[warp][w][(mt * 16 + g + (i >> 1) * 8) * COLS + 8 * r + 2 * t + (i & 1)] = acc[w][r][mt][i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int o = threadIdx.x + THREADS * i;
    if (o >= OUTS) break;
    const int64_t m = o / COLS, n = n0 + o % COLS;
    if (m >= p.M || n >= p.N) continue;
    T s[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      s[w] = part[0][w][o];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) s[w] += part[k][w][o];
    }
    float v[2] = {fmaf(static_cast<float>(s[0]) * xs[i], ws[i], b[i]), 0.0f};
    activate_all(v, p.activation);
    if constexpr (GATED) v[0] *= fmaf(static_cast<float>(s[1]) * xs[i], wus[i], bu[i]);
    store_from_f32(p.y, m * p.ld_y + n, p.out_dtype, v[0] + res[i]);
  }
}

}  // namespace glp
