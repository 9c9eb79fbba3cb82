// The paged cache in 8 bits: OCP e4m3 codes and a scale 2^(b - 127) for every 16
// rows of a page and key head, [pages, kv heads, page size / 16] bytes b.
//
// A power of two, so that a block's rows move to a larger scale by their exponents alone
// (only what falls below the least normal code is rounded again), and every code times its scale
// is a bf16 exactly: the products see what the cache holds.
#pragma once

#include "attn.h"

namespace dsk {

constexpr int kScaleRows = 16;       // rows that share a scale
// Scale bytes that are given out: from 2^-100, so that the least code (2^-9) stays a normal
// bf16, to 2^119, so that the largest (448) stays a finite one.
constexpr int kLeastScale = 27, kMostScale = 246;
constexpr float kMostCode = 448.0f;

// Least byte b in range with top <= 448 * 2^(b - 127); 448 is 1.75 * 2^8.
__device__ __forceinline__ int scale_byte(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int b = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(b, kLeastScale), kMostScale);
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// 2^(127 - b) for a byte that is given out.
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23); }

// Eight values times inv (a power of two) as codes, to nearest even.  check: some may be no finite number, an
// infinity or NaN, which are NaN then (the type has no infinity), or beyond 448, which are 448.
__device__ __forceinline__ u32x2 to_codes(const float (&x)[8], float inv, bool check) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i] * inv;
  if (check)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = fminf(fmaxf(y[i], -kMostCode), kMostCode);
      if ((__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u) y[i] = __builtin_nanf("");
    }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return u32x2{static_cast<uint32_t>(lo), static_cast<uint32_t>(hi)};
}

// Four codes times `factor` (a power of two, at most 1).
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float factor) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), true);
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * factor, a[1] * factor, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * factor, b[1] * factor, lo, true));
}
// 2^(from - to) for scale bytes from <= to.
__device__ __forceinline__ float scale_step(int from, int to) {
  return from - to < -126 ? 0.0f : __uint_as_float(static_cast<uint32_t>(127 + from - to) << 23);
}

// Four codes times a scale as bf16, exactly.
__device__ __forceinline__ u32x2 codes_to_bf16(uint32_t codes, float scale) {
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))};
}
// Bit 7 of a byte is set where the code is a NaN.
__device__ __forceinline__ uint32_t nan_codes(uint32_t codes) { return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

}  // namespace dsk
