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

__device__ __forceinline__ uint32_t magnitude_bits(float x) {
  return __float_as_uint(x) & 0x7FFFFFFFu;
}

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

// a * s, both halves at once.
__device__ __forceinline__ float2 mul2(float2 a, float2 s) {
  float2 r;
  asm("{ .reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(s.x), "f"(s.y));
  return r;
}

// 8 values times `inv` as 8 e4m3 bytes.
template <bool kAny>
__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], float inv) {
  const float2 s = make_float2(inv, inv);
  float2 p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = mul2(make_float2(v[2 * i], v[2 * i + 1]), s);
  return make_uint2(e4m3x4<kAny>(p[0].x, p[0].y, p[1].x, p[1].y),
                    e4m3x4<kAny>(p[2].x, p[2].y, p[3].x, p[3].y));
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

__device__ __forceinline__ void store8(__nv_bfloat16 *p, const Raw8<__nv_bfloat16> &r) {
  *reinterpret_cast<uint4 *>(p) = r.a;
}
__device__ __forceinline__ void store8(float *p, const Raw8<float> &r) {
  reinterpret_cast<uint4 *>(p)[0] = r.a;
  reinterpret_cast<uint4 *>(p)[1] = r.b;
}

// Elements [0, n) of the 8 at p, zeros behind them; whole aligned chunks in
// one or two 16-byte loads.
template <typename T>
__device__ __forceinline__ Raw8<T> load8_edge(const T *p, int n, bool aligned) {
  if (aligned && n >= 8) return load8(p);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? to_float<T>(p[i]) : 0.0f;
  Raw8<T> r;
  pack(v, r);
  return r;
}

template <typename T>
__device__ __forceinline__ void store8_edge(T *p, const Raw8<T> &r, int n, bool aligned) {
  if (aligned && n >= 8) {
    store8(p, r);
    return;
  }
  float v[8];
  unpack(r, v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = from_float<T>(v[i]);
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

inline bool aligned_to(const void *p, size_t pitch_bytes, size_t to) {
  return (reinterpret_cast<uintptr_t>(p) % to) == 0 && pitch_bytes % to == 0;
}

}  // namespace b128
}  // namespace cmb
