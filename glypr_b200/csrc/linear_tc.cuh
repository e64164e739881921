// glp_linear on the 5th-generation tensor cores: persistent, warp-specialised tiles of
//
//   y = act(x w^T xs ws + b) [* (x w_up^T xs wus + bu)] + residual
//
// One kernel for every operand type (kind::f16, kind::f8f6f4 with e4m3, kind::i8 with int32 sums),
// because a K step is the same 128 bytes per row for all of them.  Warp 0 loads x and w tiles by TMA
// (128-byte swizzle, K padded with the map's zero fill), warp 1 issues the MMAs into one of two
// accumulator buffers in tensor memory, and the other warps drain the other buffer: scales, bias,
// activation, gate and residual in f32, one rounding, bulk stores.
//
//   CG = 2  pairs of CTAs on 256 x 256 tiles (each CTA loads its 128 rows of x and 128 of w)
//   CG = 1  one CTA per 128 x BN tile, for products with too few 256 x 256 tiles to fill the device
//
// A gated product's tile holds BN/2 columns of w and the same BN/2 of w_up side by side, fetched from
// the two matrices as they are; a pair takes w in one CTA and w_up in the other.
//
// The residual rows come by TMA into the same 32-row x 128-byte boxes that the outputs leave from,
// and y may be the residual itself: a box is read before the same box is stored, and no other warp
// touches its elements.  Where y or residual does not suit TMA (16-byte base and pitch) the box holds
// 32 f32 columns and the warp writes them out row by row, one element per lane (26,943 x 4,055 x 161 int8
// with residual: 197 us, 130 us with 4,056 columns).
//
// What bounds it, on a B200 at its 1 kW limit: the large products draw it and run at 1.2 to 1.6 of 1.965
// GHz, so their time is their energy.  131,072 x 768 x 1,152 bf16 with bias and residual takes 235 us (990
// TFLOP/s), 178 us of it with the drain left out; 16,384 x 4,096 x 4,096 e4m3 with erf-GELU, bias and
// residual 265 us (2.07 PFLOP/s; plain 229 us); gated int8 131,072 x 1,152 x 768 240 us (1.93 POP/s), 163 us
// without the drain.  The operands' way into shared memory comes next: 32 KB per CTA and K step of 512 MMA
// cycles.  Below one wave of tiles the time is latency: launch, one load, the K steps, the drain.
//
// The drain's shape was measured: its warps must not wait for one another (a barrier per tile among 16 warps
// with common column values: 1.18 times the time on plain bf16 131,072 x 768 x 1,152; 8 warps with values of
// their own: 1.03 times glp_bf16_gemm's, which has no epilogue), must release the accumulator as soon as it
// is read (gated int8: 236 us, 252 us after the stores), and needs few instructions rather than few special
// functions (one reciprocal for two outputs: 265 us instead of 236).
#pragma once
#include "common.cuh"
#include "linear.cuh"

namespace glp {

constexpr int kMmaF16 = 0, kMmaE4M3 = 1, kMmaI8 = 2;

struct LinearTcParams {
  LinearParams a;
  int m_tiles, n_tiles, k_blocks;
  int k_step;       // elements per 128-byte K step
  uint32_t idesc;
  int tma_out;      // y (and residual) go by bulk copies
};

template <int CG, int BN, bool GATED, int EPI>
struct LinearTcCfg {
  static constexpr int OUT_N = GATED ? BN / 2 : BN;  // output columns per tile
  static constexpr int EPI_WARPS = EPI;
  static constexpr int W = 4 * OUT_N / EPI;          // output columns per epilogue warp
  static constexpr int CH = GATED && EPI == 16 ? 16 : 32;  // ... drained at a time (96 registers with 16 warps)
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int STAGES = BN == 64 ? 6 : (EPI == 16 ? 4 : 5);
  static constexpr uint32_t A_BYTES = 128 * 128;
  static constexpr uint32_t B_ROWS = CG == 2 ? BN / 2 : BN;  // rows of w (and w_up) in this CTA
  static constexpr uint32_t B_BYTES = B_ROWS * 128;
  static constexpr uint32_t TMEM_COLS = 2 * BN;
  static constexpr uint32_t BOX_OFFSET = STAGES * (A_BYTES + B_BYTES);  // one 4 KB box per epilogue warp
  // f32 [scale | bias | scale of w_up | bias_up][W] per epilogue warp
  static constexpr uint32_t COL_OFFSET = BOX_OFFSET + EPI_WARPS * 4096;
  static constexpr uint32_t COL_BYTES = (GATED ? 4 : 2) * W * 4;
  static constexpr uint32_t BAR_OFFSET = COL_OFFSET + EPI_WARPS * COL_BYTES;
  static constexpr size_t SMEM = BAR_OFFSET + 512;
  static_assert(W == 32 || W == 64 || W == 128, "whole chunks of columns per warp");
  static_assert(SMEM <= 232448, "shared memory per CTA");
};

template <int KIND, int CG>
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
#define GLP_UMMA(cg, kind)                                                                                  \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                            \
               "tcgen05.mma.cta_group::" cg ".kind::" kind " [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), \
               "l"(b), "r"(idesc), "r"(acc))
  if constexpr (CG == 1) {
    if constexpr (KIND == kMmaF16) GLP_UMMA("1", "f16");
    if constexpr (KIND == kMmaE4M3) GLP_UMMA("1", "f8f6f4");
    if constexpr (KIND == kMmaI8) GLP_UMMA("1", "i8");
  } else {
    if constexpr (KIND == kMmaF16) GLP_UMMA("2", "f16");
    if constexpr (KIND == kMmaE4M3) GLP_UMMA("2", "f8f6f4");
    if constexpr (KIND == kMmaI8) GLP_UMMA("2", "i8");
  }
#undef GLP_UMMA
}

// 16 / 32 consecutive accumulator columns, and the wait for such loads that also names their registers, so
// that no use of them is scheduled before it
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) { tmem_ld_wait_tied(r); }
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// accumulator columns -> x w^T xs ws + b, on packed f32 pairs
template <int KIND, int N>
__device__ __forceinline__ void scale_bias(const uint32_t (&r)[N], float xs, const float* sw, const float* sb,
                                           float (&v)[N]) {
  const uint64_t xs2 = f2(xs, xs);
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const float4 w = *reinterpret_cast<const float4*>(sw + j), b = *reinterpret_cast<const float4*>(sb + j);
    float a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = KIND == kMmaI8 ? static_cast<float>(static_cast<int>(r[j + i])) : u2f(r[j + i]);
    f2_split(f2_fma(f2_mul(f2(a[0], a[1]), xs2), f2(w.x, w.y), f2(b.x, b.y)), v[j], v[j + 1]);
    f2_split(f2_fma(f2_mul(f2(a[2], a[3]), xs2), f2(w.z, w.w), f2(b.z, b.w)), v[j + 2], v[j + 3]);
  }
}

// n of N elements one pitch apart, raw (zeros after the n-th), and back.  The types and the whole column
// are told apart outside the loops, so that all loads are on their way before the first is used.
template <int N>
__device__ __forceinline__ void load_column(const void* base, int64_t at, int64_t pitch, int n, bool is16, uint32_t (&v)[N]) {
  if (is16) {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if (n == N) {
#pragma unroll
      for (int i = 0; i < N; ++i, p += pitch) v[i] = *p;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i, p += pitch) v[i] = i < n ? *p : 0;
    }
  } else {
    const uint32_t* p = static_cast<const uint32_t*>(base) + at;
#pragma unroll
    for (int i = 0; i < N; ++i, p += pitch) v[i] = i < n ? *p : 0;
  }
}
template <int N>
__device__ __forceinline__ void store_column(void* base, int64_t at, int64_t pitch, int n, int dtype, const float (&v)[N]) {
  if (dtype == kF32) {
    float* p = static_cast<float*>(base) + at;
#pragma unroll
    for (int i = 0; i < N; ++i, p += pitch)
      if (i < n) *p = v[i];
    return;
  }
  uint16_t h[N];
  if (dtype == kF16) {
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = __half_as_ushort(__float2half_rn(v[i]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = __bfloat16_as_ushort(__float2bfloat16_rn(v[i]));
  }
  uint16_t* p = static_cast<uint16_t*>(base) + at;
  if (n == N) {
#pragma unroll
    for (int i = 0; i < N; ++i, p += pitch) *p = h[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i, p += pitch)
      if (i < n) *p = h[i];
  }
}

template <int KIND, int CG, int BN, bool GATED, int EPI>
__global__ void __launch_bounds__(LinearTcCfg<CG, BN, GATED, EPI>::THREADS, 1)
    linear_tc_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_u, const __grid_constant__ CUtensorMap tm_r,
                     const __grid_constant__ CUtensorMap tm_y, const LinearTcParams p) {
  using Cfg = LinearTcCfg<CG, BN, GATED, EPI>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ __align__(1024) uint8_t smem[];
  // (the same for both CTAs of a pair, so both leave before any cluster-wide step)
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) record_error(p.a.status, kErrBadArgs);
    return;
  }
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFFSET);  // of a pair: used in the leader
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;  // a pair's leader: its warps + 1 arrive forwarded from the peer
  uint64_t* drain = tempty + 2;
  uint64_t* rbar = drain + 1;    // [EPI_WARPS] residual boxes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rbar + Cfg::EPI_WARPS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* never = abort_flag + 1;  // 0: for the waits that an abort must not cut short

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int unit = CG == 2 ? static_cast<int>(cluster_id_x()) : static_cast<int>(blockIdx.x);
  const int units = CG == 2 ? static_cast<int>(n_clusters_x()) : static_cast<int>(gridDim.x);
  const int num_tiles = p.m_tiles * p.n_tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], Cfg::EPI_WARPS + (CG == 2 && leader ? 1 : 0));
    }
    mbar_init(drain, 1);
    for (int i = 0; i < Cfg::EPI_WARPS; ++i) mbar_init(&rbar[i], 1);
    *abort_flag = 0;
    *never = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (CG == 2)
    cluster_sync_all();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_launch();
  griddep_wait();  // before anything in global memory is read or written

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ TMA producer
      int s = 0;
      uint32_t ph = 0;
      int64_t loads = 0;
      for (int tile = unit; tile < num_tiles && !*abort_flag; tile += units) {
        const int m_blk = tile / p.n_tiles, n_blk = tile % p.n_tiles;
        const int row = (m_blk * CG + static_cast<int>(rank)) * 128;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1, abort_flag)) {
            record_error(p.a.status, kErrTimeoutProducer);
            *abort_flag = 1;
            break;
          }
          const int k = kb * p.k_step;
          uint8_t* a = sA + s * Cfg::A_BYTES;
          uint8_t* b = sB + s * Cfg::B_BYTES;
          if constexpr (CG == 2) {
            if (leader) mbar_arrive_expect_tx(&full[s], 2 * (Cfg::A_BYTES + Cfg::B_BYTES));
            const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
            tma_load_2d_pair(a, &tm_x, bar, k, row);
            if constexpr (GATED)
              tma_load_2d_pair(b, leader ? &tm_w : &tm_u, bar, k, n_blk * Cfg::OUT_N);
            else
              tma_load_2d_pair(b, &tm_w, bar, k, n_blk * BN + static_cast<int>(rank) * (BN / 2));
          } else {
            mbar_arrive_expect_tx(&full[s], Cfg::A_BYTES + Cfg::B_BYTES);
            tma_load_2d(a, &tm_x, &full[s], k, row);
            tma_load_2d(b, &tm_w, &full[s], k, n_blk * Cfg::OUT_N);
            if constexpr (GATED) tma_load_2d(b + Cfg::B_BYTES / 2, &tm_u, &full[s], k, n_blk * Cfg::OUT_N);
          }
          ++loads;
          if (++s == STAGES) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (*abort_flag && leader) {  // the loads still in flight land before the CTA may leave
        for (int i = 0; i < STAGES && loads > 0; ++i, --loads) {
          s = s == 0 ? STAGES - 1 : s - 1;
          if (s == STAGES - 1) ph ^= 1;
          mbar_wait(&full[s], ph, never);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ------------------------------------------------------------ MMA issuer
      int s = 0;
      uint32_t ph = 0;
      int ab = 0;
      uint32_t aph = 0;
      bool issued = false;
      for (int tile = unit; tile < num_tiles && !*abort_flag; tile += units) {
        if (!mbar_wait(&tempty[ab], aph ^ 1, abort_flag)) {
          record_error(p.a.status, kErrTimeoutMma);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(ab * BN);
        bool ok = true;
        bool ready = false;  // the next stage, probed halfway through this one's MMAs
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!ready && !mbar_wait(&full[s], ph, abort_flag)) {
            record_error(p.a.status, kErrTimeoutMma);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t ad = desc_kmajor_sw128(smem_u32(sA + s * Cfg::A_BYTES));
          const uint64_t bd = desc_kmajor_sw128(smem_u32(sB + s * Cfg::B_BYTES));
          const int s1 = s + 1 == STAGES ? 0 : s + 1;
          const uint32_t ph1 = s + 1 == STAGES ? ph ^ 1u : ph;
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // 32 bytes of K each
            umma_ss<KIND, CG>(d, ad + 2 * k, bd + 2 * k, p.idesc, (kb | k) != 0 ? 1u : 0u);
            if (k == 1) ready = kb + 1 < p.k_blocks && mbar_test_wait(&full[s1], ph1);
          }
          issued = true;
          if constexpr (CG == 2)
            umma_commit_pair_both(smem_u32(&empty[s]));
          else
            umma_commit(&empty[s]);
          s = s1;
          ph = ph1;
        }
        if (!ok) break;
        if constexpr (CG == 2)
          umma_commit_pair_both(smem_u32(&tfull[ab]));
        else
          umma_commit(&tfull[ab]);
        ab ^= 1;
        if (ab == 0) aph ^= 1;
      }
      if (issued) {  // every MMA retires before tensor memory is released
        if constexpr (CG == 2)
          umma_commit_pair(smem_u32(drain));
        else
          umma_commit(drain);
        if (!mbar_wait(drain, 0, never)) record_error(p.a.status, kErrTimeoutDrain);
      }
    } else if (CG == 2 && lane == 0) {
      // ------------------------------------------------------------ release forwarder (peer)
      const uint32_t lead_tempty = mapa_shared(smem_u32(&tempty[0]), 0);
      int ab = 0;
      uint32_t aph = 0;
      for (int tile = unit; tile < num_tiles; tile += units) {
        if (!mbar_wait(&tempty[ab], aph, abort_flag)) {
          record_error(p.a.status, kErrTimeoutEpilogue);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        tc_fence_before();
        mbar_arrive_cluster(lead_tempty + static_cast<uint32_t>(ab * sizeof(uint64_t)));
        ab ^= 1;
        if (ab == 0) aph ^= 1;
      }
    }
  } else {
    // -------------------------------------------------------------- epilogue warps
    constexpr int W = Cfg::W, CH = Cfg::CH;
    const LinearParams& a = p.a;
    const int ew = warp - 2;
    const int quad = warp & 3;  // the tensor memory lanes that this warp can read
    const int wcol = (ew >> 2) * W;
    uint8_t* box = smem + Cfg::BOX_OFFSET + ew * 4096;
    uint64_t* rb = rbar + ew;
    const bool out16 = a.out_dtype != kF32;
    const bool res_tma = p.tma_out && a.residual;
    float* col = reinterpret_cast<float*>(smem + Cfg::COL_OFFSET + ew * Cfg::COL_BYTES);
    // output columns per box: rows of 128 (16-bit, W = 32: 64) bytes
    const int slice_cols = out16 ? (W < 64 ? W : 64) : 32;
    // 16-byte chunk q of this lane's row: the swizzle of the box's tensor map
    const uint32_t row_bytes = out16 ? slice_cols * 2 : 128;
    const uint32_t row_at = lane * row_bytes, row_swz = row_bytes == 128 ? lane & 7 : (lane >> 1) & 3;
    uint32_t rph = 0;
    int ab = 0;
    uint32_t aph = 0;
    bool ok = true;
    for (int tile = unit; tile < num_tiles; tile += units) {
      const int m_blk = tile / p.n_tiles, n_blk = tile % p.n_tiles;
      const int wrow0 = (m_blk * CG + static_cast<int>(rank)) * 128 + quad * 32;
      const int row = wrow0 + lane;
      const int col0 = n_blk * Cfg::OUT_N + wcol;
      // output columns of this warp inside N, none when its rows are past M
      const int cols = wrow0 < a.M ? max(0, min(W, a.N - col0)) : 0;
      if (res_tma && lane == 0 && cols > 0) {
        bulk_wait_read_all();  // the previous tile's outputs have left the box
        mbar_arrive_expect_tx(rb, 32 * row_bytes);
        tma_load_2d(box, &tm_r, rb, col0, wrow0);
      }
      // scales and biases of this warp's columns, and of this lane's row
#pragma unroll
      for (int j = 0; j < W; j += 32) {
        const int n = col0 + j + lane;
        const bool in = n < a.N;
        col[j + lane] = a.w_scale && in ? a.w_scale[n] : 1.0f;
        col[W + j + lane] = a.bias && in ? a.bias[n] : 0.0f;
        if constexpr (GATED) {
          col[2 * W + j + lane] = a.w_up_scale && in ? a.w_up_scale[n] : 1.0f;
          col[3 * W + j + lane] = a.bias_up && in ? a.bias_up[n] : 0.0f;
        }
      }
      const float xs = a.x_scale && row < a.M ? a.x_scale[row] : 1.0f;
      __syncwarp();
      ok = __all_sync(0xffffffffu, mbar_wait(&tfull[ab], aph, abort_flag));
      if (!ok) {
        if (lane == 0 && res_tma && cols > 0) mbar_wait(rb, rph, never);
        break;
      }
      tc_fence_after();
      const uint32_t tacc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(ab * BN + wcol);
      const auto release = [&] {  // this warp has read its part of the accumulator
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[ab]);
      };
      if (cols == 0) release();
#pragma unroll 1
      for (int c = 0; c < cols; c += CH) {
        float v[CH];
        // y or residual off 16-byte rows: this lane's column of the residual's 32 rows, on its way early
        constexpr int LROWS = CH;  // 32 rows by 32 / CH lanes per column
        const int gj = lane % CH, gi = lane / CH;
        const bool gcol = c + gj < cols;
        const int grows = min(32, a.M - wrow0);
        uint32_t res[LROWS];  // raw
        if (!p.tma_out && a.residual)
          load_column<LROWS>(a.residual, (wrow0 + static_cast<int64_t>(gi)) * a.ld_residual + col0 + c + gj,
                             a.ld_residual * (32 / CH), gcol ? (grows - gi + 32 / CH - 1) / (32 / CH) : 0, out16, res);
        {
          uint32_t r[CH];
          tmem_load(tacc + c, r);
          if constexpr (GATED) {
            uint32_t u[CH];
            tmem_load(tacc + BN / 2 + c, u);
            tmem_wait(r);
            tmem_wait(u);
            if (c + CH >= cols) release();
            float vu[CH];
            scale_bias<KIND>(r, xs, col + c, col + W + c, v);
            activate_all(v, a.activation);
            scale_bias<KIND>(u, xs, col + 2 * W + c, col + 3 * W + c, vu);
#pragma unroll
            for (int j = 0; j < CH; ++j) v[j] *= vu[j];
          } else {
            tmem_wait(r);
            if (c + CH >= cols) release();
            scale_bias<KIND>(r, xs, col + c, col + W + c, v);
            activate_all(v, a.activation);
          }
        }
        if (p.tma_out) {
          const int in_slice = c % slice_cols;
          if (in_slice == 0) {  // the box: holding the residual, or free
            if (res_tma) {
              ok = __all_sync(0xffffffffu, mbar_wait(rb, rph, never));
              rph ^= 1u;
              if (!ok) break;
            } else {
              if (lane == 0) bulk_wait_read_all();
              __syncwarp();
            }
          }
          if (out16) {
#pragma unroll
            for (int q = 0; q < CH / 8; ++q) {
              uint4* at = reinterpret_cast<uint4*>(box + row_at + (((in_slice / 8 + q) ^ row_swz) << 4));
              uint32_t w[4];
              if (res_tma) {
                const uint4 o = *at;
                const uint32_t old[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  float lo, hi;
                  unpack16(old[i], a.out_dtype, lo, hi);
                  v[q * 8 + 2 * i] += lo;
                  v[q * 8 + 2 * i + 1] += hi;
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = pack16(v[q * 8 + 2 * i], v[q * 8 + 2 * i + 1], a.out_dtype);
              *at = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int q = 0; q < CH / 4; ++q) {
              float4* at = reinterpret_cast<float4*>(box + row_at + (((in_slice / 4 + q) ^ row_swz) << 4));
              const float4 o = res_tma ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
              *at = make_float4(v[4 * q] + o.x, v[4 * q + 1] + o.y, v[4 * q + 2] + o.z, v[4 * q + 3] + o.w);
            }
          }
          if (c + CH >= cols || in_slice + CH == slice_cols) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              const int slice0 = col0 + c - in_slice;
              tma_store_2d(&tm_y, box, slice0, wrow0);
              bulk_commit();
              if (res_tma && c + CH < cols) {  // one of the warp's further boxes: up to four of f32, two of 16 bits
                bulk_wait_read_all();
                mbar_arrive_expect_tx(rb, 32 * row_bytes);
                tma_load_2d(box, &tm_r, rb, slice0 + slice_cols, wrow0);
              }
            }
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int q = 0; q < CH / 4; ++q)
            *reinterpret_cast<float4*>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          __syncwarp();
          float o[LROWS];
#pragma unroll
          for (int i = 0; i < LROWS; ++i) {
            const int rr = gi + i * (32 / CH);
            o[i] = *reinterpret_cast<const float*>(box + rr * 128 + ((((gj >> 2) ^ (rr & 7)) << 4) | ((gj & 3) << 2)));
          }
          if (a.residual) {
            if (a.out_dtype == kF16) {
#pragma unroll
              for (int i = 0; i < LROWS; ++i) o[i] += __half2float(__ushort_as_half(static_cast<unsigned short>(res[i])));
            } else {
#pragma unroll
              for (int i = 0; i < LROWS; ++i) o[i] += __uint_as_float(out16 ? res[i] << 16 : res[i]);
            }
          }
          store_column<LROWS>(a.y, (wrow0 + static_cast<int64_t>(gi)) * a.ld_y + col0 + c + gj, a.ld_y * (32 / CH),
                              gcol ? (grows - gi + 32 / CH - 1) / (32 / CH) : 0, a.out_dtype, o);
        }
      }
      if (!ok) break;
      __syncwarp();  // the columns' values have been read
      ab ^= 1;
      if (ab == 0) aph ^= 1;
    }
    if (!ok && lane == 0) {
      record_error(a.status, kErrTimeoutEpilogue);
      *abort_flag = 1;
    }
    if (lane == 0) bulk_wait_all();  // this warp's stores are in global memory
  }

  // neither CTA of a pair leaves (or frees tensor memory) while the other may touch its memory
  tc_fence_before();
  if constexpr (CG == 2)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (CG == 2)
      tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
    else
      tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace glp
