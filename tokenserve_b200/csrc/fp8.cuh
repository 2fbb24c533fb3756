// The 8-bit KV cache's row format: D e4m3 codes and one float32 scale per (token, KV head) row.
//
//   scale = max(amax|x| / 448, 2^-126),  code = e4m3(x / scale),  value = code * scale
//
// 448 is e4m3's largest value, so a row uses the whole range whatever its magnitude; the floor
// keeps scale and 1 / scale normal (an all-zero row has codes 0). A row that holds an infinity or
// a NaN gets scale NaN and NaN codes: it reads back as NaN everywhere instead of as wrong numbers.
// Codes are rounded to nearest even, at most half a step (2^-4 of the value) away.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace ts {

constexpr float kE4m3Max = 448.f;

// Bits of |x|: as unsigned integers they order like the magnitudes, with NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// max(|a|, |b|, |c|), NaN if one is.
__device__ __forceinline__ float amax3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Scale of a row whose largest |x| has these bits: amax / 448, correctly rounded (a product by the
// reciprocal and one correction).
__device__ __forceinline__ float fp8_row_scale(uint32_t amax_bits) {
  constexpr float kInv = 1.f / kE4m3Max;
  const float amax = __uint_as_float(amax_bits);
  float sc = amax * kInv;
  sc = fmaxf(fmaf(fmaf(-sc, kE4m3Max, amax), kInv, sc), 0x1p-126f);
  if (amax_bits >= 0x7f800000u) sc = __uint_as_float(0x7fc00000u);
  return sc;
}

// Divides a row by its scale. With y = 1 / scale correctly rounded and q = x y, q + (x - q scale) y is
// x / scale correctly rounded (P. Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990), where the residual is exact: codes come from quotients above
// 2^-11, so scales above 2^-90 leave it 2^-124 and more. A smaller scale is taken times 2^60 with its
// row. y itself is the hardware's approximation with one such correction.
struct Fp8Divide {
  float less, inv, up;
  __device__ __forceinline__ explicit Fp8Divide(float scale) {
    up = scale < 0x1p-90f ? 0x1p60f : 1.f;
    less = -scale * up;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale * up));
    inv = fmaf(fmaf(less, inv, 1.f), inv, inv);
  }
  __device__ __forceinline__ bool small() const { return up != 1.f; }

  // Codes of a pair (low byte: a); saturating, NaN stays NaN. `a` and `b` are already times `up`.
  __device__ __forceinline__ uint32_t pair(float a, float b) const {
    const uint64_t x = two(a, b), y = two(inv, inv), q = mul2(x, y);
    const float2 f = halves(fma2(fma2(q, two(less, less), x), y, q));
    return __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
  }
  __device__ __forceinline__ uint32_t pack4(float x0, float x1, float x2, float x3) const {
    return pair(x0, x1) | pair(x2, x3) << 16;
  }
  __device__ __forceinline__ uint8_t one(float x) const { return uint8_t(pair(x * up, 0.f)); }
};

// Two codes (low half of `w`) as f16x2; exact, e4m3's values are f16 numbers.
__device__ __forceinline__ __half2 fp8_half2(uint32_t w) {
  const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
  return __half2(r);
}

__device__ __forceinline__ float fp8_float(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

}  // namespace ts
