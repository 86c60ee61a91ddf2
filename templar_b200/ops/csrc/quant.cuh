// Values in 8 bits: what the kernels that write codes and those that read them share (the format is described in quant.cu).
#pragma once
#include "common.cuh"

constexpr int QUANT_GROUP = 64;      // columns that share a scale in what a backward pass reads

struct Codes { float inv, scale; };
// From the bits of a group's largest magnitude.
static __device__ __forceinline__ Codes codes_of(uint32_t top) {
  const float a = __uint_as_float(top);
  if (top >= 0x7f800000u) return {0.f, __uint_as_float(0x7fc00000u)};
  if (a < 0x1p-100f) return {0.f, 0.f};
  return {127.f / a, a / 127.f};
}
static __device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// The largest magnitude of three, one of them a largest magnitude already; NaN where one is NaN.
static __device__ __forceinline__ float top3(float t, float x, float y) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(t), "f"(x), "f"(y));
  return r;
}

// Four codes in a word.  Added to 1.5 * 2^23, a number's last bits are its nearest whole number (ties to even, as rint) in two's
// complement: conversion instructions run at a sixteenth of the rate.  |x * inv| is at most 127 (1 + 2^-23) and never rounds to
// 128.  Multiplied and added one after the other: a fused sum would round ties of x * inv another way than rint(x * inv).
static __device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.f));
  const uint32_t w = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  return inv != 0.f ? w : 0u;        // a group that is not finite has codes of zero
}
// The codes of a word as numbers: byte b + 128 in the last place of 2^23.
static __device__ __forceinline__ void numbers4(uint32_t w, float* f) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | i)) - 8388736.f;
}

// A sum of integers times the scales of its row and its column.  The scales multiply one another first; where that leaves the normal
// numbers although the result may be one (groups are held down to 2^-100 and up to what fp32 holds), half of each scale's exponent
// waits for the end: with s = h * t and t a power of two near sqrt(s), the product h * h' and its product with the sum are normal wherever
// the result is, and a power of two changes no bit of it.  Where both ways stay normal they give the same bits.
static __device__ __forceinline__ float power_near_root(uint32_t s) { return __uint_as_float(((s >> 1) & 0x3f800000u) + 0x20000000u); }
static __device__ __forceinline__ float scaled_far(int sum, float row, float col) {
  const float tr = power_near_root(magnitude(row)), tc = power_near_root(magnitude(col));        // 2^-63 to 2^64
  const float hr = row * __uint_as_float(0x7f000000u - __float_as_uint(tr)), hc = col * __uint_as_float(0x7f000000u - __float_as_uint(tc));
  return (float)sum * (hr * hc) * fminf(tr * tc, 0x1p127f);      // 2^128 only where every sum but 0 gives infinity
}
static __device__ __forceinline__ float scaled(int sum, float row, float col) {
  const float s = row * col;
  return magnitude(s) - 0x00800000u < 0x7f000000u ? (float)sum * s : scaled_far(sum, row, col);
}
// The least and the largest magnitude of a warp's scales, zeros and what is not finite left out, and whether all their products with
// another scale are normal numbers, or zero because that one is.
struct ScaleRange { float least, most; };
static __device__ __forceinline__ ScaleRange scale_range(float s) {
  const uint32_t m = magnitude(s);
  const bool in = m - 1u < 0x7f7fffffu;
  return {__uint_as_float(__reduce_min_sync(0xffffffffu, in ? m : 0x7f800000u)), __uint_as_float(__reduce_max_sync(0xffffffffu, in ? m : 0u))};
}
static __device__ __forceinline__ bool in_range(const ScaleRange& r, float s) {
  const float m = fabsf(s);
  return m == 0.f || (m * r.least >= 0x1p-126f && m * r.most < __uint_as_float(0x7f800000u));
}
