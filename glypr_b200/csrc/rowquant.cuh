// Row kernels that write 8-bit rows with one f32 scale per row (int8 or e4m3 codes): the residual
// addition and RMS norm between two sublayers, and plain row quantisation.
//
//   x~ = x * rms(x) * post_gain   (or x),   h = (residual + x~) * layer_scalar,
//   n  = h * rms(h) * gain,   scale = max(max|n| / top, 2^-100),   code = rn(n / scale)
//
// Everything between the loads and the two roundings (h to its type, n to its code) is f32, and a row stays
// in registers from its one read to its one write.  Whole chunks of 8 elements are bound by memory: 262,144 x
// 768 (f16 + bf16 residual, both norms) 240 us = 5.9 TB/s, 131,072 x 1,152 f16 quantised 73 us = 6.2 TB/s,
// 32,768 x 4,096 norm 141 us = 6.7 TB/s (a copy: 6.5).  Rows that start anywhere take a third more
// instructions (the gains' shift, head and tail): 10,007 x 1,543 norm 29 us = 3.7 TB/s, 65,536 x 771 90 us =
// 3.9 TB/s.  Tried and slower: gains kept in registers over a block's rows (10,007 x 1,543 56 us: fewer warps),
// edge chunks read whole and masked (34 us), a shared-memory pass is not shorter in instructions.
// Operands that stand apart in their chunks go one element per load.
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
  float eps, layer_scalar, inv_H;
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

// sum of a (SUM) and NaN-keeping maximum of b (MAX) over the G threads that share a row (8 or 16 lanes, a
// warp or the block)
template <int G, bool SUM = true, bool MAX = true>
__device__ __forceinline__ void row_reduce(float& a, float& b) {
  const uint32_t lanes = G >= 32 ? 0xffffffffu : ((1u << (G & 31)) - 1) << (threadIdx.x & 31 & ~(G - 1));
#pragma unroll
  for (int o = G >= 32 ? 16 : G / 2; o > 0; o >>= 1) {
    if constexpr (SUM) a += __shfl_xor_sync(lanes, a, o);
    if constexpr (MAX) b = max_nan(b, __shfl_xor_sync(lanes, b, o));
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
      if constexpr (SUM) a += part[i].x;
      if constexpr (MAX) b = max_nan(b, part[i].y);
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

constexpr float kMaxF32 = 3.4028235e38f;

// rms(v) from the sum of squares; NaN where that is beyond f32 (values of 2^64, long before they are), for a row
// that has no norm here is not one of zeros.  (Taking such rows times a power of two instead cost rows of 2,048
// and of 16,384 elements 11 and 18 %, for its code alone: registers and the loads' order.)
__device__ __forceinline__ float inv_rms(float ss, const RowQuantParams& p) {
  const float ms = fmaf(ss, p.inv_H, p.eps);
  return ms <= kMaxF32 ? rsqrtf(ms) : __int_as_float(0x7fffffff);
}

// The factor from values to codes: top / amax by one rounded quotient (the rms and the scale's own rounding
// cancel in it), and 1 / scale where the scale is the floor.  With the quotient of the rounded rms and scale
// in its place three times as many codes fell on the other side of a rounding boundary.
__device__ __forceinline__ float code_factor(float amax, float inv, float& s, int q_dtype) {
  const bool above = s > kQuantFloor;  // (a scale of NaN: whatever the code)
  const float k = (above ? quant_top(q_dtype) : inv) / (above ? amax : s);
  // No codes where top / amax is beyond f32 (|h gain| under 2^-118 through an eps under 1e-15), rather than
  // ones of another row; and a finite factor, so that zeros keep code 0 where 1 / (rms scale) overflows.
  if (above && k > kMaxF32) s = __int_as_float(0x7fffffff);
  return fminf(k, kMaxF32);
}

// One element at a time, any alignment: G threads per row, NC elements per thread, H <= G * NC.
// NORM false: plain row quantisation.
template <int G, int NC, bool NORM>
__global__ void __launch_bounds__(G < 128 ? 128 : G) row_quant_any_kernel(const RowQuantParams p) {
  constexpr int ROWS = G < 128 ? 128 / G : 1;
  const int t = threadIdx.x % G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / G;
  griddep_launch();
  griddep_wait();
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
      inv = inv_rms(ss, p);
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
    const float inv_h = inv_rms(ss, p);
    float s = scale_of(amax * inv_h, p.q_dtype);
    const float k = code_factor(amax, inv_h, s, p.q_dtype);
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

// ---------------------------------------------------------------------------- 8 elements at a time
// The same rows in aligned chunks of 8 elements (one 16-byte load of a 16-bit row, two of an f32 row,
// one 8-byte store of codes).  Rows need not start on a chunk boundary -- a packed odd width has no two
// rows alike -- as long as x, residual, h and q all stand at the same place in their chunks: the row is
// then `head` elements up to its first boundary, whole chunks, and a tail, and the at most 14 elements of
// head and tail go one per lane beside the chunks (by element in the lane that holds the chunk they cost
// more than all the chunks: 131,072 x 250 norm 154 us).
template <int DT>
constexpr int kBytes = DT == kF32 ? 4 : 2;

template <int DT>
struct Chunk {  // 8 raw elements
  uint4 v[kBytes<DT> / 2];
};

__device__ __forceinline__ uint4 ld_stream(const void* p) {  // read once: no line in L1
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// The gains: kept in L1, for every row reads them again, by coherent loads, for the kernel is resident while the
// call before it may still write them.  Neither volatile nor tied to memory, so that they are free to move up
// among the row's loads and stores; only the pointers, made after the wait, hold them behind it.
__device__ __forceinline__ const float* after_wait(const float* p) {
  asm volatile("" : "+l"(p) : : "memory");
  return p;
}
__device__ __forceinline__ float4 ld_gain4(const float* p) {
  float4 v;
  asm("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float ld_gain(const float* p) {
  float v;
  asm("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

// elements [e, e + 8) of the row at `row`, zeros for no chunk
template <int DT>
__device__ __forceinline__ Chunk<DT> load_chunk(const uint8_t* row, int e, bool on) {
  constexpr int B = kBytes<DT>;
  Chunk<DT> c;
#pragma unroll
  for (int i = 0; i < B / 2; ++i) c.v[i] = on ? ld_stream(row + static_cast<int64_t>(e) * B + 16 * i) : make_uint4(0u, 0u, 0u, 0u);
  return c;
}

// as four packed f32 pairs
template <int DT>
__device__ __forceinline__ void chunk_f32(const Chunk<DT>& c, uint64_t (&v)[4]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&c);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == kF32) {
      v[j] = f2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
    } else if constexpr (DT == kBF16) {
      v[j] = f2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      v[j] = f2(f.x, f.y);
    }
  }
}

template <int DT>
__device__ __forceinline__ void store_chunk(uint8_t* row, int e, bool on, const uint64_t (&p)[4]) {
  constexpr int B = kBytes<DT>;
  if (!on) return;
  float v[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) f2_split(p[j], v[2 * j], v[2 * j + 1]);
  uint8_t* at = row + static_cast<int64_t>(e) * B;
  if constexpr (B == 4) {
    *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(at + 16) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == kBF16) {
        w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ void store_codes(uint8_t* row, int e, bool on, int q_dtype, const uint64_t (&p)[4], uint64_t k) {
  uint32_t w[2];
  if (q_dtype == kI8) {
    // v * k + 1.5 * 2^23 rounds once to the nearest integer, ties to even, and leaves it in the low byte
    float b[8];
    const uint64_t magic = f2(12582912.0f, 12582912.0f);
#pragma unroll
    for (int j = 0; j < 4; ++j) f2_split(f2_fma(p[j], k, magic), b[2 * j], b[2 * j + 1]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = __byte_perm(__byte_perm(__float_as_uint(b[4 * i]), __float_as_uint(b[4 * i + 1]), 0x0040),
                         __byte_perm(__float_as_uint(b[4 * i + 2]), __float_as_uint(b[4 * i + 3]), 0x0040), 0x5410);
  } else {
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float lo, hi;
      f2_split(f2_mul(p[j], k), lo, hi);
      h[j] = code_e4m3x2(lo, hi);
    }
    w[0] = __byte_perm(h[0], h[1], 0x5410);
    w[1] = __byte_perm(h[2], h[3], 0x5410);
  }
  if (on) *reinterpret_cast<uint2*>(row + e) = make_uint2(w[0], w[1]);
}

// largest magnitude of m and 8 values, keeping a NaN
__device__ __forceinline__ float max8(float m, const uint64_t (&p)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float lo, hi;
    f2_split(p[j], lo, hi);
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(lo), "f"(hi));
  }
  return m;
}

// gain[e .. e + 8), zeros for no chunk.  From an unaligned e the aligned words around it are loaded and
// shifted by e & 3, which is the same for the whole row.
template <bool SHIFTED>
__device__ __forceinline__ void load_gain(const float* gain, bool aligned16, int e, bool on, uint64_t (&p)[4]) {
  if (!on) {
    p[0] = p[1] = p[2] = p[3] = f2(0.0f, 0.0f);
    return;
  }
  const int s = SHIFTED ? e & 3 : 0;
  if (!SHIFTED || (aligned16 && s == 0)) {
    const float4 a = ld_gain4(gain + e), b = ld_gain4(gain + e + 4);
    p[0] = f2(a.x, a.y), p[1] = f2(a.z, a.w), p[2] = f2(b.x, b.y), p[3] = f2(b.z, b.w);
    return;
  }
  float v[8];
  if (aligned16) {
    float w[12];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 f = ld_gain4(gain + (e - s) + 4 * i);
      w[4 * i] = f.x, w[4 * i + 1] = f.y, w[4 * i + 2] = f.z, w[4 * i + 3] = f.w;
    }
    // (the s values that the third word is needed for; the row may end with them)
    w[8] = ld_gain(gain + (e - s + 8));
    w[9] = s > 1 ? ld_gain(gain + (e - s + 9)) : 0.0f;
    w[10] = s > 2 ? ld_gain(gain + (e - s + 10)) : 0.0f;
    w[11] = 0.0f;
    // a shift by s in two steps, so that every index is known at compile time
#pragma unroll
    for (int j = 0; j < 10; ++j) w[j] = s & 2 ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s & 1 ? w[j + 1] : w[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ld_gain(gain + e + j);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = f2(v[2 * j], v[2 * j + 1]);
}

__device__ __forceinline__ float f2_hsum(uint64_t v) {
  float lo, hi;
  f2_split(v, lo, hi);
  return lo + hi;
}

// how a row lies in its chunks: anywhere; from a chunk's start, in whole chunks; and exactly as many as
// its threads hold
constexpr int kShifted = 0, kFlush = 1, kFull = 2;

// G threads per row, NC chunks per thread: a row has at most G NC whole chunks.  XT, HT: types of x and of
// residual / h.  gains16: both gains start on 16-byte boundaries (kFlush and kFull promise it).
// A norm of 5 chunks a lane in 16-bit types needs just over the 80 registers that three blocks per SM leave
// (65,536 x 1,152, both norms: 101 us, 121 us with two).
template <int G, int NC, int XT, int HT, bool NORM>
constexpr int kRowBlocks = NORM && G == 32 && NC == 5 && kBytes<XT> == 2 && kBytes<HT> == 2 ? 3 : 0;
template <int G, int NC, int XT, int HT, bool NORM, int PLACE>
__global__ void __launch_bounds__(G <= 32 ? 256 : G, kRowBlocks<G, NC, XT, HT, NORM>) row_quant_kernel(const RowQuantParams p, bool gains16) {
  constexpr int ROWS = G <= 32 ? 256 / G : 1;
  constexpr bool SHIFTED = PLACE == kShifted;
  constexpr int ED = !SHIFTED ? 0 : (G >= 16 ? 1 : 2);  // head and tail elements per lane
  const int t = threadIdx.x % G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / G;
  griddep_launch();
  griddep_wait();
  if (row >= p.M) return;  // the row's threads together
  const uint8_t* xr = static_cast<const uint8_t*>(p.x) + row * p.ld_x * kBytes<XT>;
  uint8_t* qr = static_cast<uint8_t*>(p.q) + row * p.ld_q;
  const int off = SHIFTED ? static_cast<int>(reinterpret_cast<uintptr_t>(xr) / kBytes<XT> & 7) : 0;
  const int head = SHIFTED && off ? min(8 - off, p.H) : 0;
  const int chunks = (p.H - head) / 8;
  const auto e_of = [&](int c) { return head + (c * G + t) * 8; };
  const auto on = [&](int c) { return PLACE == kFull || c * G + t < chunks; };
  // this lane's elements of head and tail
  int ne[ED ? ED : 1];
  bool oe[ED ? ED : 1];
#pragma unroll
  for (int d = 0; d < ED; ++d) {
    const bool last = G >= 16 ? t >= 8 : d == 1;
    const int j = t & 7, from = head + chunks * 8;
    ne[d] = last ? from + j : j;
    oe[d] = t < 16 && (last ? from + j < p.H : j < head);
  }
  Chunk<XT> xc[NC];
  if constexpr (!NORM || PLACE != kFull) {
#pragma unroll
    for (int c = 0; c < NC; ++c) xc[c] = load_chunk<XT>(xr, e_of(c), on(c));
  }
  float ve[ED ? ED : 1];
#pragma unroll
  for (int d = 0; d < ED; ++d) ve[d] = oe[d] ? load_as_f32(xr, ne[d], XT) : 0.0f;
  uint64_t v[NC][4];
  float none = 0.0f, amax = 0.0f;
  if constexpr (NORM) {
    const float *post_gain = after_wait(p.post_gain), *gain = after_wait(p.gain);
    const uint8_t* rr = static_cast<const uint8_t*>(p.residual) + row * p.ld_residual * kBytes<HT>;
    uint8_t* hr = static_cast<uint8_t*>(p.h) + row * p.ld_h * kBytes<HT>;
    Chunk<HT> rc[NC];
    float re[ED ? ED : 1];
    // Full rows: x and residual side by side, for which the compiler takes more registers and keeps more in
    // flight (98,304 x 1,024 f16 and bf16 133 us, 159 us with x first; 196,608 x 512 117 / 120; f32 rows would
    // rather have x first, 243 / 223); the other kinds, whose x is on its way by now, are slower with it
    // (65,536 x 1,152: 115 us, 101 us).
    if constexpr (PLACE == kFull) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        xc[c] = load_chunk<XT>(xr, e_of(c), true);
        if (p.residual) rc[c] = load_chunk<HT>(rr, e_of(c), true);
      }
    } else if (p.residual) {
#pragma unroll
      for (int c = 0; c < NC; ++c) rc[c] = load_chunk<HT>(rr, e_of(c), on(c));
    }
    if (p.residual) {
#pragma unroll
      for (int d = 0; d < ED; ++d) re[d] = oe[d] ? load_as_f32(rr, ne[d], HT) : 0.0f;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) chunk_f32<XT>(xc[c], v[c]);
    uint64_t inv2 = f2(1.0f, 1.0f);
    if (post_gain) {
      uint64_t ss2 = f2(0.0f, 0.0f);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss2 = f2_fma(v[c][j], v[c][j], ss2);
      float ss = f2_hsum(ss2);
#pragma unroll
      for (int d = 0; d < ED; ++d) ss = fmaf(ve[d], ve[d], ss);
      row_reduce<G, true, false>(ss, none);
      const float inv = inv_rms(ss, p);
      inv2 = f2(inv, inv);
#pragma unroll
      for (int d = 0; d < ED; ++d) ve[d] = ve[d] * inv * (oe[d] ? ld_gain(post_gain + ne[d]) : 0.0f);
    }
    const uint64_t scalar2 = f2(p.layer_scalar, p.layer_scalar);
    uint64_t ss2 = f2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e = e_of(c);
      uint64_t g[4];
      if (post_gain) {
        load_gain<SHIFTED>(post_gain, gains16, e, on(c), g);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[c][j] = f2_mul(f2_mul(v[c][j], inv2), g[j]);
      }
      if (p.residual) {
        uint64_t r[4];
        chunk_f32<HT>(rc[c], r);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[c][j] = f2_add(v[c][j], r[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[c][j] = f2_mul(v[c][j], scalar2);
        ss2 = f2_fma(v[c][j], v[c][j], ss2);
      }
      if (p.h) store_chunk<HT>(hr, e, on(c), v[c]);
      if (gain) {
        load_gain<SHIFTED>(gain, gains16, e, on(c), g);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[c][j] = f2_mul(v[c][j], g[j]);
      }
      amax = max8(amax, v[c]);
    }
    float ss = f2_hsum(ss2);
#pragma unroll
    for (int d = 0; d < ED; ++d) {
      if (p.residual) ve[d] += re[d];
      ve[d] *= p.layer_scalar;
      ss = fmaf(ve[d], ve[d], ss);
      if (p.h && oe[d]) store_from_f32(hr, ne[d], HT, ve[d]);
      if (gain) ve[d] *= oe[d] ? ld_gain(gain + ne[d]) : 0.0f;
      amax = max_nan(amax, fabsf(ve[d]));
    }
    row_reduce<G, true, true>(ss, amax);
    const float inv_h = inv_rms(ss, p);
    float s = scale_of(amax * inv_h, p.q_dtype);
    const float k = code_factor(amax, inv_h, s, p.q_dtype);
    if (t == 0) p.scale[row] = s;
#pragma unroll
    for (int c = 0; c < NC; ++c) store_codes(qr, e_of(c), on(c), p.q_dtype, v[c], f2(k, k));
#pragma unroll
    for (int d = 0; d < ED; ++d)
      if (oe[d]) qr[ne[d]] = code_of(ve[d] * k, p.q_dtype);
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      chunk_f32<XT>(xc[c], v[c]);
      amax = max8(amax, v[c]);
    }
#pragma unroll
    for (int d = 0; d < ED; ++d) amax = max_nan(amax, fabsf(ve[d]));
    row_reduce<G, false, true>(none, amax);
    const float s = scale_of(amax, p.q_dtype);
    // (v * k is within an ulp of v / s; the rounded quotient, a correction more, gave no fewer codes beyond a
    // rounding boundary -- the scale itself is rounded -- and took 80 us instead of 74 for 131,072 x 1,152)
    const float k = 1.0f / s;
    if (t == 0) p.scale[row] = s;
#pragma unroll
    for (int c = 0; c < NC; ++c) store_codes(qr, e_of(c), on(c), p.q_dtype, v[c], f2(k, k));
#pragma unroll
    for (int d = 0; d < ED; ++d)
      if (oe[d]) qr[ne[d]] = code_of(ve[d] * k, p.q_dtype);
  }
}

}  // namespace glp
