// Host side of glp_norm_residual_q8 and glp_quantize_rows: argument checks, the choice of kernel,
// launches.
#include <algorithm>

#include "op_rows.cuh"

namespace {

using namespace glp::op;
using glp::RowQuantParams;

static_assert(GLP_DTYPE_F32 == glp::kF32 && GLP_DTYPE_F16 == glp::kF16 && GLP_DTYPE_BF16 == glp::kBF16 &&
              GLP_DTYPE_I8 == glp::kI8 && GLP_DTYPE_E4M3 == glp::kE4M3, "dtype codes");

// Whether every row's x, residual, h and q stand at the same place in their chunks of 8 elements.
bool same_chunks(const RowQuantParams& p) {
  const auto place = [](const void* a, int size) { return reinterpret_cast<uintptr_t>(a) / size % 8; };
  const int xs = dtype_size(p.x_dtype), hs = dtype_size(p.h_dtype);
  const uintptr_t x = place(p.x, xs);
  return place(p.q, 1) == x && (p.ld_q - p.ld_x) % 8 == 0 &&
         (!p.residual || (place(p.residual, hs) == x && (p.ld_residual - p.ld_x) % 8 == 0)) &&
         (!p.h || (place(p.h, hs) == x && (p.ld_h - p.ld_x) % 8 == 0));
}

template <bool NORM>
int launch_row_quant(const RowQuantParams& p, cudaStream_t st) {
  if (same_chunks(p)) {
    if constexpr (NORM) {
      const bool gains16 = aligned(p.gain, 16) && aligned(p.post_gain, 16);
      if (p.x_dtype == GLP_DTYPE_F32) return launch_norm_chunks<glp::kF32>(p, gains16, st);
      if (p.x_dtype == GLP_DTYPE_F16) return launch_norm_chunks<glp::kF16>(p, gains16, st);
      return launch_norm_chunks<glp::kBF16>(p, gains16, st);
    } else {
      if (p.x_dtype == GLP_DTYPE_F32) return launch_quant_chunks<glp::kF32>(p, st);
      if (p.x_dtype == GLP_DTYPE_F16) return launch_quant_chunks<glp::kF16>(p, st);
      return launch_quant_chunks<glp::kBF16>(p, st);
    }
  }
  const unsigned rows = static_cast<unsigned>(p.M);
  if (p.H <= 256) return launch(glp::row_quant_any_kernel<32, 8, NORM>, (rows + 3) / 4, 128, 0, 1, st, p);
  if (p.H <= 2048) return launch(glp::row_quant_any_kernel<128, 16, NORM>, rows, 128, 0, 1, st, p);
  if (p.H <= 8192) return launch(glp::row_quant_any_kernel<512, 16, NORM>, rows, 512, 0, 1, st, p);
  return launch(glp::row_quant_any_kernel<1024, 32, NORM>, rows, 1024, 0, 1, st, p);
}

int norm_residual_q8(const glp_norm_q8_args* a, cudaStream_t st) {
  if (!a) return fail(GLP_ERR_INVALID_ARG, "args is NULL");
  if (a->M < 0 || a->H < 1 || a->H > GLP_QUANT_MAX_H)
    return fail(GLP_ERR_INVALID_ARG, "norm needs M >= 0 and 1 <= H <= 32768");
  if (!wide_dtype(a->x_dtype) || !wide_dtype(a->h_dtype)) return fail(GLP_ERR_INVALID_ARG, "x and h must be F32, F16 or BF16");
  if (!code_dtype(a->q_dtype)) return fail(GLP_ERR_INVALID_ARG, "q must be I8 or E4M3");
  if (!(a->eps >= 0.0f)) return fail(GLP_ERR_INVALID_ARG, "eps must be >= 0");
  RowQuantParams p{};
  p.M = a->M, p.H = a->H;
  p.x = a->x, p.residual = a->residual, p.post_gain = a->post_gain, p.gain = a->gain;
  p.h = a->h, p.q = a->q, p.scale = a->scale;
  p.ld_x = a->ld_x, p.ld_residual = a->ld_residual, p.ld_h = a->ld_h, p.ld_q = a->ld_q;
  // At least the smallest normal f32: a row of zeros then keeps its zeros, and what squares lose below f32's range
  // is lost against it.
  p.eps = std::max(a->eps, 1.17549435e-38f), p.layer_scalar = a->layer_scalar, p.inv_H = static_cast<float>(1.0 / p.H);
  p.x_dtype = a->x_dtype, p.h_dtype = a->h_dtype, p.q_dtype = a->q_dtype;
  if (!pitch(&p.ld_x, p.H) || !pitch(&p.ld_residual, p.H) || !pitch(&p.ld_h, p.H) || !pitch(&p.ld_q, p.H))
    return fail(GLP_ERR_INVALID_ARG, "a row pitch is shorter than H");
  if (a->M == 0) return GLP_OK;
  if (!p.x || !p.q || !p.scale) return fail(GLP_ERR_INVALID_ARG, "null pointer");
  if (p.h && p.h == p.residual && p.ld_h != p.ld_residual)
    return fail(GLP_ERR_INVALID_ARG, "h in place of residual needs the same row pitch");
  if (!aligned(p.x, dtype_size(p.x_dtype)) || !aligned(p.residual, dtype_size(p.h_dtype)) ||
      !aligned(p.h, dtype_size(p.h_dtype)) || !aligned(p.post_gain, 4) || !aligned(p.gain, 4) || !aligned(p.scale, 4))
    return fail(GLP_ERR_INVALID_ARG, "a pointer is not aligned to its element type");
  return launch_row_quant<true>(p, st);
}

int quantize_rows(const void* x, int x_dtype, int64_t ld_x, int M, int H, void* q, int q_dtype, int64_t ld_q,
                  float* scale, cudaStream_t st) {
  if (M < 0 || H < 1 || H > GLP_QUANT_MAX_H)
    return fail(GLP_ERR_INVALID_ARG, "row quantisation needs M >= 0 and 1 <= H <= 32768");
  if (!wide_dtype(x_dtype)) return fail(GLP_ERR_INVALID_ARG, "x must be F32, F16 or BF16");
  if (!code_dtype(q_dtype)) return fail(GLP_ERR_INVALID_ARG, "q must be I8 or E4M3");
  RowQuantParams p{};
  p.M = M, p.H = H, p.x = x, p.q = q, p.scale = scale, p.ld_x = ld_x, p.ld_q = ld_q;
  p.x_dtype = x_dtype, p.q_dtype = q_dtype;
  if (!pitch(&p.ld_x, H) || !pitch(&p.ld_q, H)) return fail(GLP_ERR_INVALID_ARG, "a row pitch is shorter than H");
  if (M == 0) return GLP_OK;
  if (!x || !q || !scale) return fail(GLP_ERR_INVALID_ARG, "null pointer");
  if (!aligned(x, dtype_size(x_dtype)) || !aligned(scale, 4))
    return fail(GLP_ERR_INVALID_ARG, "a pointer is not aligned to its element type");
  return launch_row_quant<false>(p, st);
}

}  // namespace

extern "C" {

int glp_norm_residual_q8(const glp_norm_q8_args* args, void* stream) {
  return guarded([&] { return norm_residual_q8(args, static_cast<cudaStream_t>(stream)); });
}

int glp_quantize_rows(const void* x, int x_dtype, int64_t ld_x, int M, int H, void* q, int q_dtype, int64_t ld_q,
                      float* scale, void* stream) {
  return guarded([&] { return quantize_rows(x, x_dtype, ld_x, M, H, q, q_dtype, ld_q, scale, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
