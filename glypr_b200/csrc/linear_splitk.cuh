// glp_linear for products with few output tiles and a long K: a cluster of S CTAs takes one 128 x 64 tile
// (gated: 64 columns of w and the same 64 of w_up), each CTA a share of the K steps with the pipeline of
// linear_tc_kernel, and the accumulators are joined through distributed shared memory.  CTA r of the
// cluster owns columns [r 64/S, (r + 1) 64/S): every CTA stores its partial sums of those columns into
// r's shared memory, and after one cluster barrier r adds the S of them in rank order (int8: exactly, in
// int32), applies the epilogue and writes its columns.  Nothing is left in global memory between calls.
// What its columns need besides the sums is fetched before the products end: fetched after the barrier it
// cost 3 us more (768 x 768 f16, M = 128, S = 2: 9.3 us, 6.3 us).  The time is latency: 0.285 us per K step of
// a CTA on 4.6 us (gated 6.8 us) for launch, first load, exchange and stores.  300 x 8,000 f16, M = 128: 9.0 us
// with S = 8, 37.6 us unsplit (the plain bytes: 1.1 us).
#pragma once
#include "linear_tc.cuh"

namespace glp {

template <bool GATED>
struct LinearSplitCfg {
  static constexpr int BN = GATED ? 128 : 64;
  static constexpr int OUT_N = 64;
  static constexpr int THREADS = 320;
  static constexpr int STAGES = GATED ? 4 : 6;
  static constexpr uint32_t A_BYTES = 128 * 128;
  static constexpr uint32_t B_BYTES = BN * 128;
  static constexpr uint32_t PART_OFFSET = STAGES * (A_BYTES + B_BYTES);  // [w | w_up][source][row][64 / S] words
  static constexpr uint32_t BAR_OFFSET = PART_OFFSET + BN * 128 * 4;
  static constexpr size_t SMEM = BAR_OFFSET + 256;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// p.m_tiles x p.n_tiles clusters of S = 2, 4 or 8 CTAs, S <= p.k_blocks
template <int KIND, bool GATED, int S>
__global__ void __launch_bounds__(320, 1)
    linear_split_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                        const __grid_constant__ CUtensorMap tm_u, const LinearTcParams p) {
  using Cfg = LinearSplitCfg<GATED>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {  // (the same for every CTA of the cluster)
    if (threadIdx.x == 0) record_error(p.a.status, kErrBadArgs);
    return;
  }
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFFSET);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* never = abort_flag + 1;

  const LinearParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(cluster_id_x());
  const int m_blk = tile / p.n_tiles, n_blk = tile % p.n_tiles;
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * rank / S);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (rank + 1) / S);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    *abort_flag = 0;
    *never = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::BN);
    tmem_relinquish();
  }
  tc_fence_before();
  cluster_sync_all();  // every CTA of the cluster runs before any stores into another
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_launch();
  griddep_wait();  // before anything in global memory is read or written

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ TMA producer
      int s = 0, loads = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[s], ph ^ 1, abort_flag)) {
          record_error(a.status, kErrTimeoutProducer);
          *abort_flag = 1;
          break;
        }
        const int k = kb * p.k_step;
        uint8_t* b = sB + s * Cfg::B_BYTES;
        mbar_arrive_expect_tx(&full[s], Cfg::A_BYTES + Cfg::B_BYTES);
        tma_load_2d(sA + s * Cfg::A_BYTES, &tm_x, &full[s], k, m_blk * 128);
        tma_load_2d(b, &tm_w, &full[s], k, n_blk * 64);
        if constexpr (GATED) tma_load_2d(b + 64 * 128, &tm_u, &full[s], k, n_blk * 64);
        ++loads;
        if (++s == STAGES) {
          s = 0;
          ph ^= 1;
        }
      }
      if (*abort_flag) {  // the loads still in flight land before the CTA may leave
        for (int i = 0; i < STAGES && loads > 0; ++i, --loads) {
          s = s == 0 ? STAGES - 1 : s - 1;
          if (s == STAGES - 1) ph ^= 1;
          mbar_wait(&full[s], ph, never);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ------------------------------------------------------------ MMA issuer
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[s], ph, abort_flag)) {
          record_error(a.status, kErrTimeoutMma);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint64_t ad = desc_kmajor_sw128(smem_u32(sA + s * Cfg::A_BYTES));
        const uint64_t bd = desc_kmajor_sw128(smem_u32(sB + s * Cfg::B_BYTES));
#pragma unroll
        for (int k = 0; k < 4; ++k)  // 32 bytes of K each
          umma_ss<KIND, 1>(tmem_base, ad + 2 * k, bd + 2 * k, p.idesc, (kb - kb0) | k ? 1u : 0u);
        umma_commit(&empty[s]);
        if (++s == STAGES) {
          s = 0;
          ph ^= 1;
        }
      }
      umma_commit(tfull);  // also after an abort: every MMA retires before tensor memory is released
      if (!mbar_wait(tfull, 0, never)) record_error(a.status, kErrTimeoutDrain);
    }
  }

  // What this CTA's columns need besides the sums, on its way during the products: thread i of the
  // epilogue's 256 finishes 4 columns of IT rows.
  constexpr int CW = 64 / S, PER_ROW = CW / 4, IT = 128 * PER_ROW / 256, NW = GATED ? 2 : 1;
  const int et = static_cast<int>(threadIdx.x) - 64;
  const int c = et % PER_ROW * 4;
  const int64_t n = static_cast<int64_t>(n_blk) * 64 + rank * CW + c;
  float ws[NW][4], bs[NW][4], xs[IT], res[IT][4];
  if (warp >= 2) {
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* wp = w ? a.w_up_scale : a.w_scale;
      const float* bp = w ? a.bias_up : a.bias;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ws[w][j] = wp && n + j < a.N ? wp[n + j] : 1.0f;
        bs[w][j] = bp && n + j < a.N ? bp[n + j] : 0.0f;
      }
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int64_t m = static_cast<int64_t>(m_blk) * 128 + (et + 256 * it) / PER_ROW;
      xs[it] = a.x_scale && m < a.M ? a.x_scale[m] : 1.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        res[it][j] = a.residual && m < a.M && n + j < a.N ? load_as_f32(a.residual, m * a.ld_residual + n + j, a.out_dtype) : 0.0f;
    }
    // -------------------------------------------------------------- partial sums -> their owners
    const bool ok = __all_sync(0xffffffffu, mbar_wait(tfull, 0, never));
    if (!ok && lane == 0) {
      record_error(a.status, kErrTimeoutEpilogue);
      *abort_flag = 1;
    }
    if (ok) {
      tc_fence_after();
      const int quad = warp & 3, half = (warp - 2) >> 2;
      const uint32_t tacc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * 32;
      const uint32_t part = smem_u32(smem + Cfg::PART_OFFSET);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        uint32_t r[32];
        tmem_ld32(tacc + w * 64, r);
        tmem_ld_wait_tied(r);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const int col = half * 32 + j;
          const uint32_t at = part + (((w * S + rank) * 128 + quad * 32 + lane) * CW + col % CW) * 4;
          st_cluster_v4(mapa_shared(at, static_cast<uint32_t>(col / CW)), r[j], r[j + 1], r[j + 2], r[j + 3]);
        }
      }
      tc_fence_before();
    }
  }

  __syncwarp();
  cluster_sync_all();  // every CTA's sums are in their owners' shared memory
  if (warp >= 2 && !*abort_flag) {
    const float* part = reinterpret_cast<const float*>(smem + Cfg::PART_OFFSET);
    const size_t os = a.out_dtype == kF32 ? 4 : 2;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int r = (et + 256 * it) / PER_ROW;
      const int64_t m = static_cast<int64_t>(m_blk) * 128 + r;
      if (m >= a.M || n >= a.N) continue;
      float v[NW][4];
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float* at = part + ((w * S) * 128 + r) * CW + c;
        if constexpr (KIND == kMmaI8) {
          int4 t = *reinterpret_cast<const int4*>(at);
#pragma unroll
          for (int k = 1; k < S; ++k) {
            const int4 u = *reinterpret_cast<const int4*>(at + k * 128 * CW);
            t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
          }
          v[w][0] = static_cast<float>(t.x), v[w][1] = static_cast<float>(t.y);
          v[w][2] = static_cast<float>(t.z), v[w][3] = static_cast<float>(t.w);
        } else {
          float4 t = *reinterpret_cast<const float4*>(at);
#pragma unroll
          for (int k = 1; k < S; ++k) {
            const float4 u = *reinterpret_cast<const float4*>(at + k * 128 * CW);
            t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
          }
          v[w][0] = t.x, v[w][1] = t.y, v[w][2] = t.z, v[w][3] = t.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[w][j] = fmaf(v[w][j] * xs[it], ws[w][j], bs[w][j]);
        if (w == 0) activate_all(v[0], a.activation);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[0][j] = (GATED ? v[0][j] * v[NW - 1][j] : v[0][j]) + res[it][j];
      const int64_t yi = m * a.ld_y + n;
      uint8_t* y = static_cast<uint8_t*>(a.y) + yi * os;
      if (n + 4 <= a.N && (reinterpret_cast<uintptr_t>(y) & (4 * os - 1)) == 0) {
        if (os == 4)
          *reinterpret_cast<float4*>(y) = make_float4(v[0][0], v[0][1], v[0][2], v[0][3]);
        else
          *reinterpret_cast<uint2*>(y) = make_uint2(pack16(v[0][0], v[0][1], a.out_dtype), pack16(v[0][2], v[0][3], a.out_dtype));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < a.N) store_from_f32(a.y, yi + j, a.out_dtype, v[0][j]);
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::BN);
  }
}

}  // namespace glp
