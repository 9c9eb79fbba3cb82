// Shared pieces of the attention kernels (norm and rotation, prompts, the paged cache).
#pragma once

#include "tile.h"

namespace dsk {

// A value that a row does not see must not reach it, and its weight of zero times
// an infinity or a NaN would.  Where the rows of a tile see different keys, values
// are checked first: bit 15 (31) of nonfinite_bits is set where the low (high)
// bf16 is infinite or NaN (an exponent of ones carries into the sign's place).
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t two) {
  return ((two & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
// The two bf16, zero in the place of infinities and NaN.
__device__ __forceinline__ uint32_t finite_only(uint32_t two) {
  const uint32_t b = nonfinite_bits(two);
  return two & ~((b >> 15) * 0xffffu);
}
// An infinity or NaN itself, zero for a finite bf16.
__device__ __forceinline__ float nonfinite_only(uint16_t v) {
  return (v & 0x7f80u) == 0x7f80u ? bf16_bits_to_f32(v) : 0.0f;
}

// The paged cache as kernels see it.
struct CacheView {
  uint16_t* k;
  uint16_t* v;
  const int32_t* table;
  int64_t table_stride;
  int32_t n_pages, page_shift, n_seqs, max_pages;   // page size 2^page_shift
};

inline int page_shift_of(int page_size) { return __builtin_ctz(static_cast<unsigned>(page_size)); }

inline CacheView cache_view(const dsk_kv_cache& c, void* k, void* v, const int32_t* table) {
  return CacheView{static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), table, c.table_stride,
                   c.n_pages, page_shift_of(c.page_size), c.n_seqs, c.max_pages};
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_huge_valf();

// Two floats as bf16, rounded to nearest even (one instruction on gfx950).
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
  return __builtin_bit_cast(uint32_t, v);
}

// c + lo + hi of a pair of bf16, in float32 (one instruction on gfx950).
__device__ __forceinline__ float add_bf16_pair(uint32_t two, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), bf16x2{static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)}, c, false);
}

// max / sum with the lane 32 (16) lanes away, in one instruction each.
__device__ __forceinline__ float max_across32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_across16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What a call has beside the plain ones' arguments: positions on several axes (axis: of each pair), the
// tokens' rows in the cache, the cache's scales and its keys' weights.
struct QkMore {
  const int32_t *axis = nullptr, *rows = nullptr;
  int64_t axis_stride = 0;
  int32_t n_axes = 1;
  uint8_t *k_scale = nullptr, *v_scale = nullptr;
  float* key_weights = nullptr;
};
hipError_t launch_qk(const dsk_qk_desc& d, const void* q, const void* k, const void* v, const int32_t* positions,
                     const int32_t* seq, const double* freq, const float* q_gamma, const float* k_gamma,
                     const CacheView* cache, const QkMore& more, void* q_out, void* k_out,
                     hipStream_t s);   // cache: null, no append

// What a decode step's cache has beside its rows (f8: scales, weigh: its keys' weights).
struct PagedMore {
  bool f8 = false, weigh = false;
  const uint8_t *k_scale = nullptr, *v_scale = nullptr;
  float* key_weights = nullptr;
};
// Workspace of dsk_paged_attention, in bytes.
size_t paged_workspace(const dsk_paged_desc& d, const dsk_kv_cache& c, const PagedMore& more);
hipError_t launch_paged(const dsk_paged_desc& d, const dsk_kv_cache& c, const PagedMore& more, const void* q, const CacheView& view,
                        const int32_t* lens, const int32_t* prefix, void* out, void* ws, hipStream_t s);
// Workspace of dsk_kv_evict, in bytes (codes: a cache in 8 bits).
size_t evict_workspace(const dsk_evict_desc& d, const dsk_kv_cache& c, bool codes);
hipError_t launch_evict(const dsk_evict_desc& d, const dsk_kv_cache& c, const CacheView& view, uint8_t* k_scale, uint8_t* v_scale,
                        float* weights, const int32_t* lens, int32_t* lens_out, void* ws, hipStream_t s);
hipError_t launch_prompt(const dsk_prompt_desc& d, const void* q, const void* k, const void* v, const int32_t* cu_q,
                         const int32_t* cu_k, void* out, hipStream_t s);

}  // namespace dsk
