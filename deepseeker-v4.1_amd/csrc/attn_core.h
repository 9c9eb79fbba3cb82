// Query rows against a run of keys with both products on 32x32x16 MFMAs, the
// building block of prompt attention and of a shared prefix.
//
// A workgroup of NW waves holds 32 NW query rows, 32 a wave; every 64 keys and
// values are brought to LDS once for all of them (global_load_lds: no registers
// in between), two buffers deep.  As in the paged kernel, S^T = K q^T leaves a
// query row in every lane (column lane & 31) and its keys 8 a + 4 h + b in the
// registers 4 a + b of lane half h = lane >> 5, which is the B operand of
// O^T = V^T p^T for the key order {16 s + 4 h + 0..3, 16 s + 8 + 4 h + 0..3}: p stays in its lane,
// and so do the maximum, the sum and the rescaling of a row.  V^T, the A
// operand, comes from LDS with transposing reads (four keys by 16 elements in
// every 16 lanes).
//
// LDS rows are the keys' D elements in 16-byte chunks.  K: chunk c of row r at
// c ^ (r & (D / 8 - 1)), so 8 rows at one chunk (a fragment read) fall on 8
// different bank groups.  V: a transposing read of 32 lanes takes 4 chunks of 4
// rows; exclusive-or with 4 (r & 3) (D 128) or 4 ((r >> 1) & 1) (D 64: two rows
// side by side in the banks) spreads those 16 pieces over all banks.
#pragma once

#include "attn.h"

namespace dsk {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kFlKeys = 64;          // keys of a tile

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ void dma16(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// Every load of this wave has landed and its LDS reads are complete, then the workgroup barrier.
__device__ __forceinline__ void wait_all_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int D>
__device__ __forceinline__ int swz_k(int r) { return r & (D / 8 - 1); }
template <int D>
__device__ __forceinline__ int swz_v(int r) { return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }

// Four keys (16-lane groups: rows) of 16 elements, transposed: lane i of 16 gets element i of the four.
__device__ __forceinline__ u32x2 read_tr(const char* p) {
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
  return __builtin_bit_cast(u32x2, r);
}

// State of a wave's 32 rows: lane l holds row l & 31; register 4 a + b of o[dt]
// is element 32 dt + 8 a + 4 (l >> 5) + b; l is this lane half's part of the sum.
template <int D>
struct FlashRows {
  f32x16 o[D / 32];
  float m, l;
};

template <int D>
constexpr int flash_lds() { return 2 * 2 * kFlKeys * D * 2; }

// Tiles [t0, t1) of 64 keys; q[ks]: the lane's row, elements 16 ks + 8 (lane >> 5) .. +8;
// lim: the last key that the lane's row sees, w_min / w_max: least and largest lim of
// the wave's rows (wave-uniform); b_min: least lim of the workgroup's rows.  rows(tile, wave's first row in it, &k, &v, &ks, &vs, &last): pointers
// to that row of K and V, their strides, and the last row after it that may be read.
template <int D, int NW, class Rows>
__device__ __forceinline__ void flash(const bf16x8 (&q)[D / 16], int t0, int t1, int lim, int w_min, int w_max,
                                      int b_min, float c2, char* lds, Rows rows, FlashRows<D>& st) {
  constexpr int CH = D / 8, RPI = 64 / CH, WR = kFlKeys / NW, NI = WR / RPI, KS = D / 16;
  constexpr int kTile = kFlKeys * D * 2;
  static_assert(NI >= 1, "every wave loads whole instructions");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hf = lane >> 5;

  auto issue = [&](int t, int buf) {
    const uint16_t *kp, *vp;
    int64_t ks, vs;
    int last;
    rows(t, wave * WR, kp, vp, ks, vs, last);
    char* kd = lds + buf * 2 * kTile + wave * WR * D * 2;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = i * RPI + lane / CH, rr = min(r, last);
      const int row = wave * WR + r;
      dma16(kp + rr * ks + 8 * ((lane % CH) ^ swz_k<D>(row)), kd + i * RPI * D * 2);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = i * RPI + lane / CH, rr = min(r, last);
      const int row = wave * WR + r;
      dma16(vp + rr * vs + 8 * ((lane % CH) ^ swz_v<D>(row)), kd + kTile + i * RPI * D * 2);
    }
  };

  if (t0 < t1) issue(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    wait_all_barrier();
    if (t + 1 < t1) issue(t + 1, buf ^ 1);
    const char* kl = lds + buf * 2 * kTile;
    const char* vl = kl + kTile;
    // some rows see a part of the tile only: are all of its values finite?
    bool finite = true;
    if (t * kFlKeys + kFlKeys - 1 > b_min) {
      uint32_t bits = 0;
#pragma unroll
      for (int i = threadIdx.x; i < kTile / 16; i += 64 * NW) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(vl + 16 * i);
        bits |= nonfinite_bits(x[0]) | nonfinite_bits(x[1]) | nonfinite_bits(x[2]) | nonfinite_bits(x[3]);
      }
      finite = !__syncthreads_or(bits);
    }
    if (t * kFlKeys > w_max) continue;               // keys that none of the wave's rows sees
    f32x16 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = f32x16{};
      const int row = 32 * kt + n;
      const char* kr = kl + row * D * 2;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[kt] = mfma32(as_bf16x8(*reinterpret_cast<const u32x4*>(kr + 16 * ((2 * ks + hf) ^ swz_k<D>(row)))), q[ks], s[kt]);
    }
    if (t * kFlKeys + kFlKeys - 1 > w_min) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t * kFlKeys + 32 * kt + 8 * (i >> 2) + 4 * hf + (i & 3) > lim) s[kt][i] = kNegInf;
    }
    float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(fmaxf(top, s[0][i]), s[1][i]);
    top = max_across32(top) * c2;
    if (__any(top > st.m)) {
      const float mn = fmaxf(st.m, top);
      const float f = st.m == mn ? 1.0f : __builtin_amdgcn_exp2f(st.m - mn);
      st.m = mn;
      st.l *= f;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) st.o[dt] *= f;
    }
    const float mu = st.m == kNegInf ? 0.0f : st.m;
    bf16x8 p[4];
#pragma unroll
    for (int s4 = 0; s4 < 4; ++s4) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(s[s4 >> 1][8 * (s4 & 1) + i] * c2 - mu);
        st.l += e[i];
      }
      // p to bf16: relative 2^-9 each, of random sign over the keys, next to the
      // output's own rounding of 2^-9
      p[s4] = as_bf16x8(u32x4{pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7])});
    }
    const int l16 = lane & 15;
    if (!finite) {
      // rarely: the product of the finite values, and the others to the rows that see them
#pragma unroll 1
      for (int key = 0; key < kFlKeys; ++key) {
        const bool sees = t * kFlKeys + key <= lim;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int d = 32 * dt + 8 * (i >> 2) + 4 * hf + (i & 3);
            const float x = nonfinite_only(*reinterpret_cast<const uint16_t*>(
                vl + key * D * 2 + 16 * ((d >> 3) ^ swz_v<D>(key)) + 2 * (d & 7)));
            st.o[dt][i] += sees ? x : 0.0f;
          }
      }
    }
#pragma unroll
    for (int s4 = 0; s4 < 4; ++s4) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const int r0 = 16 * s4 + 4 * hf + (l16 >> 2);
        const int c = 4 * dt + 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
        const u32x2 lo = read_tr(vl + r0 * D * 2 + 16 * (c ^ swz_v<D>(r0)) + 8 * (l16 & 1));
        const u32x2 hi = read_tr(vl + (r0 + 8) * D * 2 + 16 * (c ^ swz_v<D>(r0 + 8)) + 8 * (l16 & 1));
        u32x4 w{lo[0], lo[1], hi[0], hi[1]};
        if (!finite)
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = finite_only(w[i]);
        st.o[dt] = mfma32(as_bf16x8(w), p[s4], st.o[dt]);
      }
    }
  }
}

// Splits of a shared prefix over workgroups, and its pass over all of the batch's rows.
int prefix_splits(int64_t rows, int kv_heads, int prefix_len);
hipError_t launch_prefix(const dsk_paged_desc& d, const void* q, const dsk_kv_cache& c, const int32_t* prefix,
                         int splits, float* pre_o, float* pre_ml, hipStream_t s);

}  // namespace dsk
