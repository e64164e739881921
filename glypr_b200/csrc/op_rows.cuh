// The launches of row_quant_kernel for one type of x; each op_rows_*.cu instantiates one.
#pragma once
#include "operators.h"
#include "rowquant.cuh"

namespace glp {
namespace op {

template <int XT>
int launch_norm_chunks(const RowQuantParams& p, bool gains16, cudaStream_t st);
template <int XT>
int launch_quant_chunks(const RowQuantParams& p, cudaStream_t st);

#ifdef GLP_ROWS_XT

// Rows that fill their threads' chunks exactly take the form without checks, in every shape but that of 1,024
// threads: 262,144 x 256 norm 78 us, 85 us with checks, 12,288 x 8,192 132 / 144, 196,608 x 512 quantised 46 / 52,
// 131,072 x 768 47 / 52 (its norm 141 / 136, the one shape with 98,304 x 1,024, 134 / 132, that loses); 32,768
// elements of 1,024 threads, f32 norm 841 / 431: 64 registers do not hold its loads.
template <int G, int NC, int XT, int HT, bool NORM, int PLACE>
int launch_chunks(const RowQuantParams& p, bool gains16, cudaStream_t st) {
  if constexpr (PLACE == kFlush && G < 1024) {
    if (p.H == 8 * G * NC) return launch_chunks<G, NC, XT, HT, NORM, kFull>(p, gains16, st);
  }
  constexpr int ROWS = G <= 32 ? 256 / G : 1;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(p.M) + ROWS - 1) / ROWS);
  return launch(row_quant_kernel<G, NC, XT, HT, NORM, PLACE>, grid, G <= 32 ? 256 : G, 0, 1, st, p, gains16);
}

// The fewest lanes whose chunks stay few: 8 up to 256 elements (262,144 x 64 norm 25 us, 41 us with 16 lanes,
// 262,144 x 160 65 us, 81 us with a warp), 16 up to 512, a warp up to 1,280; past that 128 threads: 32,768 x
// 2,008 bf16 with both norms 85 us, 122 us with a warp per row; row quantisation, which holds half as much,
// 32,768 x 1,537 27 us with a warp (128 threads took a fifth more).  Wider rows take the smallest block whose chunks
// they fill: 32,768 x 5,000 quantisation 73 us, 170 us with 512 threads of 2 chunks.
template <int XT, int HT, bool NORM, int PLACE>
int launch_width(const RowQuantParams& p, int chunks, bool gains16, cudaStream_t st) {
  if (chunks <= 8) return launch_chunks<8, 1, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 16) return launch_chunks<8, 2, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 32) return launch_chunks<8, 4, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 64) return launch_chunks<16, 4, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 96) return launch_chunks<32, 3, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 128) return launch_chunks<32, 4, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 160) return launch_chunks<32, 5, XT, HT, NORM, PLACE>(p, gains16, st);
  if constexpr (!NORM) {
    if (chunks <= 192) return launch_chunks<32, 6, XT, HT, NORM, PLACE>(p, gains16, st);
    if (chunks <= 224) return launch_chunks<32, 7, XT, HT, NORM, PLACE>(p, gains16, st);
  }
  if (chunks <= 256) return launch_chunks<128, 2, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 384) return launch_chunks<128, 3, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 512) return launch_chunks<128, 4, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 640) return launch_chunks<128, 5, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 768) return launch_chunks<256, 3, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 1024) return launch_chunks<256, 4, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 1536) return launch_chunks<512, 3, XT, HT, NORM, PLACE>(p, gains16, st);
  if (chunks <= 2048) return launch_chunks<512, 4, XT, HT, NORM, PLACE>(p, gains16, st);
  return launch_chunks<1024, 4, XT, HT, NORM, PLACE>(p, gains16, st);
}

template <int XT, int HT, bool NORM>
int launch_place(const RowQuantParams& p, bool gains16, cudaStream_t st) {
  const int chunks = p.H / 8;
  const bool flush = reinterpret_cast<uintptr_t>(p.x) / dtype_size(p.x_dtype) % 8 == 0 && p.ld_x % 8 == 0 && p.H % 8 == 0;
  if (!flush || !gains16) return launch_width<XT, HT, NORM, kShifted>(p, chunks, gains16, st);
  return launch_width<XT, HT, NORM, kFlush>(p, chunks, gains16, st);
}

template <int XT>
int launch_norm_chunks(const RowQuantParams& p, bool gains16, cudaStream_t st) {
  if (p.h_dtype == kF32) return launch_place<XT, kF32, true>(p, gains16, st);
  if (p.h_dtype == kF16) return launch_place<XT, kF16, true>(p, gains16, st);
  return launch_place<XT, kBF16, true>(p, gains16, st);
}
template <int XT>
int launch_quant_chunks(const RowQuantParams& p, cudaStream_t st) {
  return launch_place<XT, XT, false>(p, true, st);
}

template int launch_norm_chunks<GLP_ROWS_XT>(const RowQuantParams&, bool, cudaStream_t);
template int launch_quant_chunks<GLP_ROWS_XT>(const RowQuantParams&, cudaStream_t);

#endif  // GLP_ROWS_XT

}  // namespace op
}  // namespace glp
