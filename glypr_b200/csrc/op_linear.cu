// Host side of glp_linear: argument checks, the choice of kernel, tensor maps, launches.
#include <algorithm>
#include <atomic>

#include "linear_any.cuh"
#include "linear_rows.cuh"
#include "linear_splitk.cuh"
#include "linear_tc.cuh"
#include "operators.h"

namespace {

using namespace glp::op;
using glp::LinearParams;

static_assert(GLP_ACT_NONE == glp::kActNone && GLP_ACT_RELU == glp::kActRelu && GLP_ACT_SILU == glp::kActSilu &&
              GLP_ACT_GELU_TANH == glp::kActGeluTanh && GLP_ACT_GELU_ERF == glp::kActGeluErf, "activation codes");

template <int DT>
int launch_any(const LinearParams& p, cudaStream_t st) {
  const int64_t tiles = ((p.M + 63ll) / 64) * ((p.N + 63ll) / 64);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(tiles, 1 << 20));
  return launch(p.w_up ? glp::linear_any_kernel<DT, true> : glp::linear_any_kernel<DT, false>, grid, 256, 0, 1, st, p);
}

// ------------------------------------------------------------------------------ tensor-core product
// a row-major [rows, cols] matrix in boxes of box_rows rows x 128 or 64 bytes, swizzled by as many,
// zeros outside.  Encoded on every call: a map is a function of these arguments alone.
int make_map(CUtensorMap* m, const void* base, int dtype, int64_t rows, int64_t cols, int64_t ld, int box_rows,
             int box_bytes = 128) {
  const glp::EncodeTiledFn fn = glp::tensor_map_encoder();
  if (!fn) return fail(GLP_ERR_CUDA, "cuTensorMapEncodeTiled unavailable (driver too old?)");
  const int size = dtype_size(dtype);
  const CUtensorMapDataType type = size == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                               : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * size)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_bytes / size), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = fn(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return GLP_OK;
  glp::set_last_error("cuTensorMapEncodeTiled failed: " + std::to_string(r));
  return GLP_ERR_CUDA;
}

struct DeviceInfo {
  int dev, sms;
  int* status;
};

int device_info(DeviceInfo* d) {
  static std::atomic<int> sms[64];
  if (cudaGetDevice(&d->dev) != cudaSuccess || d->dev < 0 || d->dev >= 64)
    return fail(GLP_ERR_CUDA, "no usable CUDA device");
  d->sms = sms[d->dev].load(std::memory_order_relaxed);
  if (!d->sms) {
    if (cudaDeviceGetAttribute(&d->sms, cudaDevAttrMultiProcessorCount, d->dev) != cudaSuccess || d->sms < 1)
      return fail(GLP_ERR_CUDA, "cannot read the device's SM count");
    sms[d->dev].store(d->sms, std::memory_order_relaxed);
  }
  return glp::kernel_status_word(d->dev, &d->status);
}

// Instruction descriptor: f32 (int8: s32) accumulator, both operands K-major, m x n.
uint32_t mma_idesc(int dtype, int m, int n) {
  const uint32_t acc = dtype == GLP_DTYPE_I8 ? 2u : 1u;                                   // s32 | f32
  const uint32_t ab = (dtype == GLP_DTYPE_BF16 || dtype == GLP_DTYPE_I8) ? 1u : 0u;  // bf16, s8 | f16, e4m3
  return acc << 4 | ab << 7 | ab << 10 | static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}

// raises a kernel's shared-memory limit once per device
template <class K>
int raise_smem(K kernel, size_t smem, int dev, std::atomic<uint64_t>* ready) {
  const uint64_t bit = 1ull << dev;
  if (ready->load(std::memory_order_relaxed) & bit) return GLP_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return launched(e);
  ready->fetch_or(bit, std::memory_order_relaxed);
  return GLP_OK;
}

template <int KIND, int CG, int BN, bool GATED, int EPI = 8>
int launch_tc(glp::LinearTcParams p, const DeviceInfo& d, cudaStream_t st) {
  using Cfg = glp::LinearTcCfg<CG, BN, GATED, EPI>;
  const auto kernel = glp::linear_tc_kernel<KIND, CG, BN, GATED, EPI>;
  static std::atomic<uint64_t> ready{0};
  if (int rc = raise_smem(kernel, Cfg::SMEM, d.dev, &ready)) return rc;
  const LinearParams& a = p.a;
  p.m_tiles = (a.M + 128 * CG - 1) / (128 * CG);
  p.n_tiles = (a.N + Cfg::OUT_N - 1) / Cfg::OUT_N;
  p.k_step = 128 / dtype_size(a.dtype);
  p.k_blocks = (a.K + p.k_step - 1) / p.k_step;
  p.idesc = mma_idesc(a.dtype, 128 * CG, BN);
  const size_t os = dtype_size(a.out_dtype);
  p.tma_out = aligned(a.y, 16) && a.ld_y * os % 16 == 0 &&
              (!a.residual || (aligned(a.residual, 16) && a.ld_residual * os % 16 == 0));
  // rows of w (and of w_up) that one load brings: a gated single CTA takes half of each
  const int w_rows = CG == 2 ? BN / 2 : Cfg::OUT_N;
  CUtensorMap mx, mw, mu, mr, my;
  if (int rc = make_map(&mx, a.x, a.dtype, a.M, a.K, a.ld_x, 128)) return rc;
  if (int rc = make_map(&mw, a.w, a.dtype, a.N, a.K, a.ld_w, w_rows)) return rc;
  mu = mr = my = mw;
  if (GATED)
    if (int rc = make_map(&mu, a.w_up, a.dtype, a.N, a.K, a.ld_w, w_rows)) return rc;
  if (p.tma_out) {
    const int out_bytes = os == 2 && Cfg::W == 32 ? 64 : 128;
    if (int rc = make_map(&my, a.y, a.out_dtype, a.M, a.N, a.ld_y, 32, out_bytes)) return rc;
    if (a.residual)
      if (int rc = make_map(&mr, a.residual, a.out_dtype, a.M, a.N, a.ld_residual, 32, out_bytes)) return rc;
  }
  const int units = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(p.m_tiles) * p.n_tiles, d.sms / CG));
  return launch(kernel, static_cast<unsigned>(units * CG), Cfg::THREADS, Cfg::SMEM, CG, st, mx, mw, mu, mr, my, p);
}

template <int KIND, bool GATED, int S>
int launch_split(glp::LinearTcParams p, const DeviceInfo& d, cudaStream_t st) {
  using Cfg = glp::LinearSplitCfg<GATED>;
  const auto kernel = glp::linear_split_kernel<KIND, GATED, S>;
  static std::atomic<uint64_t> ready{0};
  if (int rc = raise_smem(kernel, Cfg::SMEM, d.dev, &ready)) return rc;
  const LinearParams& a = p.a;
  p.m_tiles = (a.M + 127) / 128;
  p.n_tiles = (a.N + 63) / 64;
  p.k_step = 128 / dtype_size(a.dtype);
  p.k_blocks = (a.K + p.k_step - 1) / p.k_step;
  p.idesc = mma_idesc(a.dtype, 128, Cfg::BN);
  CUtensorMap mx, mw, mu;
  if (int rc = make_map(&mx, a.x, a.dtype, a.M, a.K, a.ld_x, 128)) return rc;
  if (int rc = make_map(&mw, a.w, a.dtype, a.N, a.K, a.ld_w, 64)) return rc;
  mu = mw;
  if (GATED)
    if (int rc = make_map(&mu, a.w_up, a.dtype, a.N, a.K, a.ld_w, 64)) return rc;
  return launch(kernel, static_cast<unsigned>(p.m_tiles * p.n_tiles * S), Cfg::THREADS, Cfg::SMEM, S, st, mx, mw, mu, p);
}

template <int KIND>
int launch_tc_kind(const LinearParams& a, const DeviceInfo& d, cudaStream_t st) {
  glp::LinearTcParams p{};
  p.a = a;
  p.a.status = d.status;
  const bool gated = a.w_up != nullptr;
  // The kernel by estimated time: a fixed part, and per wave of tiles the K steps (128 bytes of a row each)
  // or, with few of them, the drain.  Microseconds in a CUDA graph, read off M = 65 .. 16,384 against N x K of
  // 768 x 768 f16, 768 x 1,152 and 2,304 x 768 int8, 4,096 x 4,096 e4m3, 2,048 x 2,048 bf16 and 300 x 8,000 f16
  // with bias and residual, and gated 1,152 x 768 int8 and x 4,096 bf16.  768 x 768 f16: M = 512: 64-wide 6.5,
  // 128-wide 8.2, pairs 11; M = 4,096: 15, 12.9, 12.  Splitting K over clusters of 2, 4, 8 (one wave of them,
  // fewer than SMs since a cluster stays within a GPC): 300 x 8,000 f16, M = 128: 37.6 unsplit, 22.3, 13.0,
  // 9.0; 4,096 x 4,096 e4m3, M = 128: 12.1, 9.7 with 2.
  const int steps = (a.K * dtype_size(a.dtype) + 127) / 128;
  const auto estimate = [&](int64_t rows, int64_t cols, int64_t slots, double fixed, double step, double drain) {
    const int64_t tiles = ((a.M + rows - 1) / rows) * ((a.N + cols - 1) / cols);
    return fixed + static_cast<double>((tiles + slots - 1) / slots) * std::max(step * steps, drain);
  };
  const double pair = estimate(256, gated ? 128 : 256, d.sms / 2, 5.0, 0.43, gated ? 3.5 : 5.4);
  const double single128 = estimate(128, gated ? 64 : 128, d.sms, 3.2, 0.37, gated ? 2.5 : 3.15);
  const double single64 = gated ? 1e30 : estimate(128, 64, d.sms, 2.9, 0.29, 2.0);
  const int64_t tiles64 = ((a.M + 127ll) / 128) * ((a.N + 63ll) / 64);
  int split = 1;
  double best = std::min({pair, single128, single64});
  for (const int S : {2, 4, 8}) {
    const int64_t room = S == 2 ? d.sms : S == 4 ? d.sms * 7 / 8 : d.sms * 3 / 4;
    const double t = (gated ? 6.8 : 4.6) + (S == 8 ? 0.4 : 0.0) + 0.285 * ((steps + S - 1) / S);
    if (tiles64 * S <= room && steps >= 2 * S && t < best) {
      best = t;
      split = S;
    }
  }
  switch (split) {
    case 2: return gated ? launch_split<KIND, true, 2>(p, d, st) : launch_split<KIND, false, 2>(p, d, st);
    case 4: return gated ? launch_split<KIND, true, 4>(p, d, st) : launch_split<KIND, false, 4>(p, d, st);
    case 8: return gated ? launch_split<KIND, true, 8>(p, d, st) : launch_split<KIND, false, 8>(p, d, st);
    default: break;
  }
  if (pair <= single128 && pair <= single64) {
    // 16 warps drain a tile whose outputs take two exponentials or reciprocals each: their phases (tensor
    // memory, special functions, stores) then overlap between warps.  131,072 x 2,304 x 768 e4m3 with SiLU:
    // 310 us, 373 us with 8; without an activation 281 us, 279 us with 8, and bf16 227 / 216 us.
    const bool heavy = a.activation == GLP_ACT_SILU || a.activation == GLP_ACT_GELU_TANH || a.activation == GLP_ACT_GELU_ERF;
    if (gated) return launch_tc<KIND, 2, 256, true, 16>(p, d, st);
    return heavy ? launch_tc<KIND, 2, 256, false, 16>(p, d, st) : launch_tc<KIND, 2, 256, false, 8>(p, d, st);
  }
  if (gated) return launch_tc<KIND, 1, 128, true>(p, d, st);
  return single128 < single64 ? launch_tc<KIND, 1, 128, false>(p, d, st) : launch_tc<KIND, 1, 64, false>(p, d, st);
}

// ------------------------------------------------------------------------------ few rows
template <int DT, bool GATED, int MT, int R, int U, int WARPS>
int launch_rows(const LinearParams& p, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>((p.N + 8ll * R - 1) / (8 * R));
  return launch(glp::linear_rows_kernel<DT, GATED, MT, R, U, WARPS>, grid, 32 * WARPS, 0, 1, st, p);
}

// Whether the few-rows kernel is the faster one: always up to 16 rows.  Its blocks each read x again, so
// with more rows only while that stays small: M = 64, 768 x 768 f16 4.9 us (tensor-memory kernel 7.3 us,
// 9 MB of x read), 4,096 x 4,096 f16 31 us (14 us, 268 MB).  Up to 32 rows also where the weights have
// too few rows for the other kernel's 64-wide tiles to fill the device (4,096 x 4,096 f16: 11 us, 14 us;
// 8,191 x 4,096 e4m3: 20 us, 17 us).  (In a CUDA graph, operands in L2, as all times of this file.)
bool few_rows(const LinearParams& p, const DeviceInfo& d) {
  if (p.M <= 16) return true;
  if (p.M > 64) return false;
  const int64_t x_traffic = (p.N + 7ll) / 8 * p.M * p.K * dtype_size(p.dtype);
  return x_traffic <= (32 << 20) || (p.M <= 32 && p.N < 48 * d.sms);
}

// R: 8 rows of w per block while those blocks fit the device at once, 16 beyond (4,096 x 4,096 f16, one row:
// 9.8 us with 8, 6.1 us with 16; 768 x 768: 2.1 / 2.6 us).
template <int DT, bool GATED>
int launch_rows(const LinearParams& p, const DeviceInfo& d, cudaStream_t st) {
  if (p.M <= 16)
    return p.N <= 16 * d.sms ? launch_rows<DT, GATED, 1, 1, 2, 16>(p, st) : launch_rows<DT, GATED, 1, 2, 2, 16>(p, st);
  if (p.M <= 32) {
    if constexpr (GATED)
      return launch_rows<DT, true, 2, 1, 1, 16>(p, st);
    else
      return p.N <= 8 * d.sms ? launch_rows<DT, false, 2, 1, 2, 16>(p, st) : launch_rows<DT, false, 2, 2, 1, 16>(p, st);
  }
  return launch_rows<DT, GATED, 4, 1, 1, GATED ? 8 : 16>(p, st);  // gated: sums of 16 warps would not fit
}

template <int DT>
int launch_rows(const LinearParams& p, const DeviceInfo& d, cudaStream_t st) {
  return p.w_up ? launch_rows<DT, true>(p, d, st) : launch_rows<DT, false>(p, d, st);
}

bool tc_operands(const LinearParams& p) {
  const size_t es = dtype_size(p.dtype);
  return aligned(p.x, 16) && aligned(p.w, 16) && aligned(p.w_up, 16) && p.ld_x * es % 16 == 0 && p.ld_w * es % 16 == 0;
}

int linear(const glp_linear_args* a, cudaStream_t st) {
  if (!a) return fail(GLP_ERR_INVALID_ARG, "args is NULL");
  if (a->M < 0 || a->N < 1 || a->K < 1) return fail(GLP_ERR_INVALID_ARG, "linear needs M >= 0, N >= 1, K >= 1");
  if (a->M > 1 << 30 || a->N > 1 << 30 || a->K > 1 << 28)  // indices of rows and bytes of a row stay in 31 bits
    return fail(GLP_ERR_INVALID_ARG, "linear needs M and N <= 2^30, K <= 2^28");
  if (a->dtype < GLP_DTYPE_F16 || a->dtype > GLP_DTYPE_E4M3)
    return fail(GLP_ERR_INVALID_ARG, "operands must be F16, BF16, I8 or E4M3");
  if (!wide_dtype(a->out_dtype)) return fail(GLP_ERR_INVALID_ARG, "y must be F32, F16 or BF16");
  if (a->activation < GLP_ACT_NONE || a->activation > GLP_ACT_GELU_ERF)
    return fail(GLP_ERR_INVALID_ARG, "unknown activation");
  if (a->dtype == GLP_DTYPE_I8 && a->K > 131071)
    return fail(GLP_ERR_INVALID_ARG, "int8 operands need K <= 131071 (int32 sums)");
  if (!a->w_up && (a->w_up_scale || a->bias_up))
    return fail(GLP_ERR_INVALID_ARG, "w_up_scale and bias_up need w_up");
  LinearParams p{};
  p.M = a->M, p.N = a->N, p.K = a->K;
  p.dtype = a->dtype, p.out_dtype = a->out_dtype, p.activation = a->activation;
  p.x = a->x, p.w = a->w, p.w_up = a->w_up, p.ld_x = a->ld_x, p.ld_w = a->ld_w;
  p.x_scale = a->x_scale, p.w_scale = a->w_scale, p.w_up_scale = a->w_up_scale;
  p.bias = a->bias, p.bias_up = a->bias_up;
  p.residual = a->residual, p.y = a->y, p.ld_residual = a->ld_residual, p.ld_y = a->ld_y;
  if (!pitch(&p.ld_x, p.K) || !pitch(&p.ld_w, p.K)) return fail(GLP_ERR_INVALID_ARG, "a row pitch is shorter than K");
  if (!pitch(&p.ld_residual, p.N) || !pitch(&p.ld_y, p.N)) return fail(GLP_ERR_INVALID_ARG, "a row pitch is shorter than N");
  if (a->M == 0) return GLP_OK;
  if (!p.x || !p.w || !p.y) return fail(GLP_ERR_INVALID_ARG, "null pointer");
  if (p.residual && p.residual == p.y && p.ld_residual != p.ld_y)
    return fail(GLP_ERR_INVALID_ARG, "y in place of residual needs the same row pitch");
  const size_t es = dtype_size(p.dtype), os = dtype_size(p.out_dtype);
  if (!aligned(p.x, es) || !aligned(p.w, es) || !aligned(p.w_up, es) || !aligned(p.y, os) || !aligned(p.residual, os) ||
      !aligned(p.x_scale, 4) || !aligned(p.w_scale, 4) || !aligned(p.w_up_scale, 4) || !aligned(p.bias, 4) ||
      !aligned(p.bias_up, 4))
    return fail(GLP_ERR_INVALID_ARG, "a pointer is not aligned to its element type");
  if (tc_operands(p)) {
    DeviceInfo d;
    if (int rc = device_info(&d)) return rc;
    if (few_rows(p, d)) {
      switch (p.dtype) {
        case GLP_DTYPE_F16: return launch_rows<glp::kF16>(p, d, st);
        case GLP_DTYPE_BF16: return launch_rows<glp::kBF16>(p, d, st);
        case GLP_DTYPE_I8: return launch_rows<glp::kI8>(p, d, st);
        default: return launch_rows<glp::kE4M3>(p, d, st);
      }
    }
    if (p.dtype == GLP_DTYPE_I8) return launch_tc_kind<glp::kMmaI8>(p, d, st);
    if (p.dtype == GLP_DTYPE_E4M3) return launch_tc_kind<glp::kMmaE4M3>(p, d, st);
    return launch_tc_kind<glp::kMmaF16>(p, d, st);
  }
  switch (p.dtype) {
    case GLP_DTYPE_F16: return launch_any<glp::kF16>(p, st);
    case GLP_DTYPE_BF16: return launch_any<glp::kBF16>(p, st);
    case GLP_DTYPE_I8: return launch_any<glp::kI8>(p, st);
    default: return launch_any<glp::kE4M3>(p, st);
  }
}

}  // namespace

extern "C" {

int glp_linear(const glp_linear_args* args, void* stream) {
  return guarded([&] { return linear(args, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
