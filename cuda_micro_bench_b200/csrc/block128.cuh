// block128.cuh — the block-scaled e4m3 form shared by the quantiser, the
// RMS norm and the GEMM: one E8M0 scale byte for each block of 128 values
// (or 128 x 128), and 8-value chunks of bf16 or fp32 rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "cmb_device.cuh"

namespace cmb {
namespace b128 {

constexpr int kBlock = 128;
constexpr float kMaxFinite = 3.40282346638528859811704183484516925e+38f;

__host__ __device__ constexpr int groups_of(int n) { return (n + kBlock - 1) / kBlock; }

// |x| where x is finite, 0 where it is not: what a block's scale is taken from.
__device__ __forceinline__ float finite_magnitude(float x) {
  const float a = fabsf(x);
  return a <= kMaxFinite ? a : 0.0f;
}

// E8M0 byte of the smallest power of two s with amax / s <= 448.  With amax =
// 1.m * 2^(E - 127) and 448 = 1.75 * 2^8 that is 2^(E - 127 - 8), or twice
// that where 1.m > 1.75; integers on the bits, so every path (quantiser,
// norm, host) agrees on a block that ends exactly at 448 * 2^n.  Under
// 2^-127 there is no E8M0 value: those blocks keep byte 0 and lose nothing,
// since amax / 2^-127 is then under 448.
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  if (amax == 0.0f) return 127u;
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 0));
}

// 2^(127 - byte), the exact reciprocal of a scale that scale_byte made (its
// bytes reach 247, so the result is a normal number).
__device__ __forceinline__ float scale_reciprocal(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);
}

// Magnitudes compare like their bits, so a maximum is an integer one, and one
// look at it tells whether a block has anything that is not finite.
constexpr uint32_t kInfBits = 0x7F800000u;

// Four values to e4m3 (nearest even), the first in the low byte.  The scale
// keeps finite values within 448, so saturation only ever meets infinities;
// where a block may hold any (kAny), those become NaN, as NaN does.
template <bool kAny>
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t q;
  asm("{ .reg .b16 l, h;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
      "mov.b32 %0, {l, h}; }"
      : "=r"(q)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  if constexpr (kAny) {
    const float v[4] = {a, b, c, d};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(fabsf(v[i]) <= kMaxFinite)) q = (q & ~(0xFFu << (8 * i))) | (0x7Fu << (8 * i));
  }
  return q;
}

// The larger magnitude; NaN wins.
__device__ __forceinline__ float max_magnitude(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// 8 values times `inv` as 8 e4m3 bytes.
template <bool kAny>
__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], float inv) {
  return make_uint2(e4m3x4<kAny>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                    e4m3x4<kAny>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
}
// The rare form, out of the way of the other.
static __device__ __noinline__ uint2 e4m3x8_any(float4 a, float4 b, float inv) {
  const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  return e4m3x8<true>(v, inv);
}

// Both bf16 halves of a word times a bf16 each (given as fp32 bits' upper
// half), in fp32: one instruction a value, with no unpacking.
__device__ __forceinline__ float2 mul_bf16x2(uint32_t w, uint32_t lo_scale, uint32_t hi_scale) {
  float2 r;
  asm("{ .reg .b16 l, h, s, t, x;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "mov.b32 {x, s}, %3;\n\t"
      "mov.b32 {x, t}, %4;\n\t"
      "fma.rn.f32.bf16 %0, l, s, %5;\n\t"
      "fma.rn.f32.bf16 %1, h, t, %5; }"
      : "=f"(r.x), "=f"(r.y)
      : "r"(w), "r"(lo_scale), "r"(hi_scale), "f"(-0.0f));
  return r;
}

// ------------------------------------------------- rows of bf16 or fp32

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// 8 consecutive elements as they lie in memory.
template <typename T>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
};
template <>
struct Raw8<float> {
  uint4 a, b;
};

__device__ __forceinline__ Raw8<__nv_bfloat16> load8(const __nv_bfloat16 *p) {
  return {*reinterpret_cast<const uint4 *>(p)};
}
__device__ __forceinline__ Raw8<float> load8(const float *p) {
  return {reinterpret_cast<const uint4 *>(p)[0], reinterpret_cast<const uint4 *>(p)[1]};
}

__device__ __forceinline__ void unpack(const Raw8<__nv_bfloat16> &r, float (&v)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack(const Raw8<float> &r, float (&v)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}

// The larger magnitudes of two pairs of bf16; NaN wins.
__device__ __forceinline__ uint32_t max_magnitude2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 v = __hmax2_nan(__habs2(*reinterpret_cast<const __nv_bfloat162 *>(&a)),
                                       __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&b)));
  return *reinterpret_cast<const uint32_t *>(&v);
}

// Largest magnitude's bits (as fp32 bits) of the 8; NaN and infinities count.
__device__ __forceinline__ uint32_t top_bits(const Raw8<__nv_bfloat16> &r) {
  const uint32_t v = max_magnitude2(max_magnitude2(r.a.x, r.a.y), max_magnitude2(r.a.z, r.a.w));
  return max(v << 16, v & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t top_bits(const Raw8<float> &r) {
  const uint32_t m = 0x7FFFFFFFu;
  return max(max(max(r.a.x & m, r.a.y & m), max(r.a.z & m, r.a.w & m)),
             max(max(r.b.x & m, r.b.y & m), max(r.b.z & m, r.b.w & m)));
}

// The same for each row and each column of 8 x 8 values.
__device__ __forceinline__ void tops(const Raw8<__nv_bfloat16> (&r)[8], uint32_t (&rmax)[8],
                                     uint32_t (&cmax)[8]) {
  uint32_t c[4] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w[4] = {r[i].a.x, r[i].a.y, r[i].a.z, r[i].a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = max_magnitude2(c[k], w[k]);
    const uint32_t v = max_magnitude2(max_magnitude2(w[0], w[1]), max_magnitude2(w[2], w[3]));
    rmax[i] = max(v << 16, v & 0xFFFF0000u);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    cmax[2 * k] = c[k] << 16;
    cmax[2 * k + 1] = c[k] & 0xFFFF0000u;
  }
}
__device__ __forceinline__ void tops(const Raw8<float> (&r)[8], uint32_t (&rmax)[8],
                                     uint32_t (&cmax)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) cmax[j] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w[8] = {r[i].a.x, r[i].a.y, r[i].a.z, r[i].a.w,
                           r[i].b.x, r[i].b.y, r[i].b.z, r[i].b.w};
    rmax[i] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t m = w[j] & 0x7FFFFFFFu;
      rmax[i] = max(rmax[i], m);
      cmax[j] = max(cmax[j], m);
    }
  }
}

__device__ __forceinline__ uint32_t bf16x2_bits(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// a * b + c of both bf16 halves, in fp32: an instruction a value, with no
// unpacking.
__device__ __forceinline__ void fma_bf16x2(uint32_t a, uint32_t b, float &c0, float &c1) {
  asm("{ .reg .b16 l, h, s, t;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "mov.b32 {s, t}, %3;\n\t"
      "fma.rn.f32.bf16 %0, l, s, %0;\n\t"
      "fma.rn.f32.bf16 %1, h, t, %1; }"
      : "+f"(c0), "+f"(c1)
      : "r"(a), "r"(b));
}

// c += a * b, element for element (exact products where both are bf16).
__device__ __forceinline__ void fma8(const Raw8<__nv_bfloat16> &a, const Raw8<__nv_bfloat16> &b,
                                     float (&c)[8]) {
  fma_bf16x2(a.a.x, b.a.x, c[0], c[1]);
  fma_bf16x2(a.a.y, b.a.y, c[2], c[3]);
  fma_bf16x2(a.a.z, b.a.z, c[4], c[5]);
  fma_bf16x2(a.a.w, b.a.w, c[6], c[7]);
}
template <typename A, typename B>
__device__ __forceinline__ void fma8(const Raw8<A> &a, const Raw8<B> &b, float (&c)[8]) {
  float u[8], v[8];
  unpack(a, u);
  unpack(b, v);
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = fmaf(u[j], v[j], c[j]);
}
// The product alone; -0 leaves its sign.
template <typename A, typename B>
__device__ __forceinline__ void mul8(const Raw8<A> &a, const Raw8<B> &b, float (&c)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = -0.0f;
  fma8(a, b, c);
}

// a + b.
__device__ __forceinline__ void add8(const Raw8<__nv_bfloat16> &a, const Raw8<__nv_bfloat16> &b,
                                     float (&c)[8]) {
  const uint32_t one = 0x3F803F80u;
  const Raw8<__nv_bfloat16> ones = {make_uint4(one, one, one, one)};
  mul8(a, ones, c);
  fma8(b, ones, c);
}
__device__ __forceinline__ void add8(const Raw8<float> &a, const Raw8<float> &b, float (&c)[8]) {
  float u[8], v[8];
  unpack(a, u);
  unpack(b, v);
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = u[j] + v[j];
}

// Rounded (nearest even) to the type of the row.
__device__ __forceinline__ void pack(const float (&v)[8], Raw8<__nv_bfloat16> &r) {
  r.a = make_uint4(bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3]), bf16x2_bits(v[4], v[5]),
                   bf16x2_bits(v[6], v[7]));
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw8<float> &r) {
  r.a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                   __float_as_uint(v[3]));
  r.b = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]),
                   __float_as_uint(v[7]));
}

template <typename T>
__device__ __forceinline__ Raw8<T> packed(const float (&v)[8]) {
  Raw8<T> r;
  pack(v, r);
  return r;
}

__device__ __forceinline__ void store8(__nv_bfloat16 *p, const Raw8<__nv_bfloat16> &r) {
  *reinterpret_cast<uint4 *>(p) = r.a;
}
__device__ __forceinline__ void store8(float *p, const Raw8<float> &r) {
  reinterpret_cast<uint4 *>(p)[0] = r.a;
  reinterpret_cast<uint4 *>(p)[1] = r.b;
}

template <typename T>
__device__ __forceinline__ void words_of(const Raw8<T> &r, uint32_t (&w)[sizeof(T) * 2]) {
  w[0] = r.a.x, w[1] = r.a.y, w[2] = r.a.z, w[3] = r.a.w;
  if constexpr (sizeof(T) == 4) w[4] = r.b.x, w[5] = r.b.y, w[6] = r.b.z, w[7] = r.b.w;
}
template <typename T>
__device__ __forceinline__ Raw8<T> from_words(const uint32_t *w) {
  Raw8<T> r;
  r.a = make_uint4(w[0], w[1], w[2], w[3]);
  if constexpr (sizeof(T) == 4) r.b = make_uint4(w[4], w[5], w[6], w[7]);
  return r;
}

// out[i] = the 4 bytes at byte `m` (0-15) + 4 i of the words in.
template <int N>
__device__ __forceinline__ void from_byte(uint32_t (&in)[N + 4], uint32_t m, uint32_t (&out)[N]) {
#pragma unroll
  for (int step = 2; step > 0; step >>= 1)
#pragma unroll
    for (int i = 0; i + step < N + 4; ++i) in[i] = (m >> 2) & step ? in[i + step] : in[i];
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(in[i], in[i + 1], 8 * (m & 3));
}

// Where a matrix begins and ends.  Chunks of rows at odd addresses are cut out
// of the aligned 16-byte pieces around them, which has to stay inside.
struct Bounds {
  uintptr_t begin, end;
  template <typename T>
  static __device__ __forceinline__ Bounds of(const T *p, size_t ld, int rows, int cols) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(p);
    return {b, b + (static_cast<size_t>(rows - 1) * ld + cols) * sizeof(T)};
  }
};

// Elements [0, n) of the 8 at byte m of the aligned 16-byte pieces around them,
// zeros behind them.
template <typename T>
struct Pieces8 {
  static constexpr int kWords = sizeof(T) * 2, kPieces = kWords / 4 + 1;
  uint4 piece[kPieces];

  __device__ __forceinline__ Raw8<T> cut(uint32_t m, int n) const {
    constexpr int N = kWords;
    uint32_t in[N + 4], w[N];
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const uint4 v = piece[k];
      in[4 * k] = v.x, in[4 * k + 1] = v.y, in[4 * k + 2] = v.z, in[4 * k + 3] = v.w;
    }
    from_byte<N>(in, m, w);
    if (n < 8) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int left = n * static_cast<int>(sizeof(T)) - 4 * i;  // bytes of this word
        if (left < 4) w[i] = left > 0 ? w[i] & ((1u << (8 * left)) - 1) : 0u;
      }
    }
    return from_words<T>(w);
  }
};

// The same one element at a time.
template <typename T>
__device__ __forceinline__ Raw8<T> load_elements(const T *p, int n) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? to_float<T>(p[i]) : 0.0f;
  Raw8<T> r;
  pack(v, r);
  return r;
}

// Elements [0, n) of the 8 at p, zeros behind them.
template <typename T>
__device__ __forceinline__ Raw8<T> load8_any(const T *p, int n, const Bounds &in) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p), piece = at & ~uintptr_t(15);
  if (n <= 0) return Raw8<T>{};
  if (at == piece && n >= 8) return load8(p);
  if (piece >= in.begin && piece + 16 * Pieces8<T>::kPieces <= in.end) {
    Pieces8<T> c;
#pragma unroll
    for (int k = 0; k < Pieces8<T>::kPieces; ++k)
      c.piece[k] = reinterpret_cast<const uint4 *>(piece)[k];
    return c.cut(static_cast<uint32_t>(at - piece), n);
  }
  return load_elements(p, n);
}

// load8_any in two steps with no branch in the first, so that many fetches are on
// their way before the first is cut to size.
template <typename T>
struct Fetch8 {
  Pieces8<T> pieces;
  bool edge;  // a piece goes past the matrix

  __device__ __forceinline__ Fetch8(const T *p, int n, const Bounds &in) : edge(false) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), first = at & ~uintptr_t(15);
    const uintptr_t end = at + min(n, 8) * sizeof(T);
#pragma unroll
    for (int k = 0; k < Pieces8<T>::kPieces; ++k) {
      const uintptr_t piece = first + 16 * k;
      const bool wanted = n > 0 && piece < end;
      const bool there = piece >= in.begin && piece + 16 <= in.end;
      pieces.piece[k] = make_uint4(0, 0, 0, 0);
      if (wanted && there) pieces.piece[k] = *reinterpret_cast<const uint4 *>(piece);
      edge |= wanted && !there;
    }
  }
  Fetch8() = default;
  __device__ __forceinline__ Raw8<T> get(const T *p, int n) const {
    if (edge) return load_elements(p, n);
    return pieces.cut(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15), n);
  }
};

template <typename T>
__device__ __forceinline__ void store_elements(T *p, const Raw8<T> &r, int from, int to) {
  float v[8];
  unpack(r, v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i >= from && i < to) p[i] = from_float<T>(v[i]);
}

// Writes elements [0, n) of the 8 to p.  The whole warp, whose lanes have
// consecutive chunks: where they do not start on 16 bytes, a lane takes the end
// of the chunk before its own from its neighbour and writes the aligned pieces.
template <typename T>
__device__ __forceinline__ void store8_any(T *p, const Raw8<T> &r, int n) {
  constexpr int N = sizeof(T) * 2;  // words
  const uint32_t m = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
  if (m == 0) {  // the same in all lanes
    if (n >= 8) store8(p, r);
    else store_elements(p, r, 0, n);
    return;
  }
  const int lane = threadIdx.x & 31;
  uint32_t w[N], c[N + 4], out[N];
  words_of(r, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __shfl_up_sync(0xffffffffu, w[N - 4 + i], 1);
#pragma unroll
  for (int i = 0; i < N; ++i) c[4 + i] = w[i];
  const uint32_t fulls = __ballot_sync(0xffffffffu, n >= 8);
  from_byte<N>(c, 16 - m, out);
  if (n < 8) {
    store_elements(p, r, 0, n);
    return;
  }
  const bool joins = lane > 0 && (fulls >> (lane - 1)) & 1;
  const bool next = lane < 31 && (fulls >> (lane + 1)) & 1;
  uint4 *piece = reinterpret_cast<uint4 *>(reinterpret_cast<uintptr_t>(p) - m);
  const int head = static_cast<int>((16 - m) / sizeof(T));
  const int tail = 8 - static_cast<int>(m / sizeof(T));
  if (joins) piece[0] = make_uint4(out[0], out[1], out[2], out[3]);
  else store_elements(p, r, 0, head);
  if constexpr (N == 8) piece[1] = make_uint4(out[4], out[5], out[6], out[7]);
  if (!next) store_elements(p, r, tail, 8);
}

// 8 bytes, or the first n of them; the odd case out of the way of the other.
static __device__ __noinline__ void store_bytes_edge(uint8_t *p, uint2 q, int n) {
  for (int i = 0; i < 8 && i < n; ++i)
    p[i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
}
__device__ __forceinline__ void store_bytes(uint8_t *p, uint2 q, int n, bool aligned) {
  if (aligned && n >= 8) *reinterpret_cast<uint2 *>(p) = q;
  else store_bytes_edge(p, q, n);
}

// ------------------------------------------------------------ host checks

// Rows and columns stay far enough under 2^31 that an index one tile or one
// round of CTAs past the end is still an int.
constexpr int kMostExtent = 0x7FFF0000;

inline bool aligned_to(const void *p, size_t pitch_bytes, size_t to) {
  return (reinterpret_cast<uintptr_t>(p) % to) == 0 && pitch_bytes % to == 0;
}

}  // namespace b128
}  // namespace cmb
