// Query rows against a run of keys with both products on 32x32x16 MFMAs, the
// building block of prompt attention and of a shared prefix.
//
// NW waves hold 32 NW query rows, 32 a wave; every 64 keys and values are brought
// to LDS once for all of them (global_load_lds: no registers in between), two
// buffers deep.  As in the paged kernel, S^T = K q^T leaves a
// query row in every lane (column lane & 31) and its keys 8 a + 4 h + b in the
// registers 4 a + b of lane half h = lane >> 5, which is the B operand of
// O^T = V^T p^T for the key order {16 s + 4 h + 0..3, 16 s + 8 + 4 h + 0..3}: p stays in its lane,
// and so do the maximum, the sum and the rescaling of a row.  V^T, the A
// operand, comes from LDS with transposing reads (four keys by 16 elements in
// every 16 lanes).
//
// A wave's tile of heads of 128 is 32 products of 32 cycles (16 for heads of 64) and about 140
// vector instructions, an exponential, a multiply-add and half a maximum, rounding and sum for every score,
// that issue between them; both pipes together bound it: 0.84 us a tile where a wave has its
// SIMD to itself, 0.92 for two tiles of two waves (64: 0.6 either way).  That is 1.07 to 1.16
// PFLOP/s over 8192 causal tokens of 32 heads (a library product of 8192^3: 1.23).  32 rows a
// wave, since 64 halve the reads of LDS but spill with heads of 128 and take the same time a row
// with 64.
//
// LDS rows are the keys' D elements in 16-byte chunks.  K: chunk c of row r at
// c ^ (r & (D / 8 - 1)), so 8 rows at one chunk (a fragment read) fall on 8
// different bank groups.  V: a transposing read of 32 lanes takes 4 chunks of 4
// rows; exclusive-or with 4 (r & 3) (D 128) or 4 ((r >> 1) & 1) (D 64: two rows
// side by side in the banks) spreads those 16 pieces over all banks.
#pragma once

#include "kv8.h"

namespace dsk {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kFlKeys = 64;          // keys of a tile

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 16 bytes a lane from base + off (bytes) to LDS at `lds` + 16 lane (both uniform).  Written
// out, since the compiler makes every later transposing read wait for all loads in
// flight when it knows that they go to LDS; the loops wait by themselves
// (wait_barrier), and the load has no result register.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is reserved, and is clobbered
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) const void*)(p))));
}
template <typename T>
__device__ __forceinline__ const T* uniform_ptr(const T* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  // readfirstlane gives an int: through 32 bits without a sign
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(v))));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(v >> 32))));
  return reinterpret_cast<const T*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// Every load of this wave has landed and its LDS reads are complete, then the
// workgroup barrier.
__device__ __forceinline__ void wait_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

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
// is element 32 dt + 8 a + 4 (l >> 5) + b; l is this lane half's part of the sum of the weights as the product uses
// them, exact (kExact alone) of the weights themselves, for those who divide other weights by it.
template <int D>
struct FlashRows {
  f32x16 o[D / 32];
  float m, l, exact;
};

constexpr int kFlBuffers = 2;        // tiles of K and of V in LDS

template <int D>
constexpr int flash_lds() { return 2 * kFlBuffers * kFlKeys * D * 2 + 16; }   // and two flags

// Tiles [t0, t1) of 64 keys; q[ks]: the lane's row, elements 16 ks + 8 (lane >> 5) .. +8;
// lim: the last key that the lane's row sees, w_min: least lim of
// the wave's rows (wave-uniform); b_min: least lim of the workgroup's rows.  rows(tile,
// wave's first row in it, &k, &v, &last): that row of K and V (the last of all where it
// lies behind) and how many rows after it may be read; kstride, vstride: elements from row to row,
// below 2^26.
//
// KH 2: two waves for 32 rows, with the lower and the upper 32 keys of every tile
// (half = wave / (NW / 2); add_halves joins them).
template <int D, int NW, int KH, bool kExact = false, class Rows>
__device__ __forceinline__ void flash(const bf16x8 (&q)[D / 16], int t0, int t1, int lim, int w_min, int b_min,
                                      float c2, char* lds, int64_t kstride, int64_t vstride, Rows rows, FlashRows<D>& st) {
  // wave-uniform by their meaning: in scalar registers
  t0 = __builtin_amdgcn_readfirstlane(t0);
  t1 = __builtin_amdgcn_readfirstlane(t1);
  w_min = __builtin_amdgcn_readfirstlane(w_min);
  b_min = __builtin_amdgcn_readfirstlane(b_min);
  constexpr int CH = D / 8, RPI = 64 / CH, WR = kFlKeys / NW, NI = WR / RPI, KS = D / 16;
  constexpr int kTile = kFlKeys * D * 2, NS = kFlBuffers, KT = 2 / KH;   // KT: a wave's 32-key parts of a tile
  static_assert(NI >= 1 && RPI % 4 == 0, "every wave loads whole instructions");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hf = lane >> 5;
  const int key0 = KH == 2 ? 32 * (wave / (NW / 2)) : 0;   // the wave's first key in a tile
  if (t0 >= t1) return;

  // LDS: K of tile t0 + j at j mod NS, then V likewise (from the first tile, so that an
  // unrolled loop knows its addresses)
  const uint32_t ldsw = lds_address(lds) + wave * WR * D * 2;
  // K (V) of tile t; rows past the last one: the last one again
  auto issue_k = [&](int t) {
    const uint16_t *kp, *vp;
    int last;
    rows(t, wave * WR, kp, vp, last);
    kp = uniform_ptr(kp);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = i * RPI + lane / CH;
      const uint32_t rr = min(r, last);
      dma16(kp, 2 * (rr * static_cast<uint32_t>(kstride) + 8 * ((lane % CH) ^ swz_k<D>(wave * WR + r))),
            ldsw + ((t - t0) % NS) * kTile + i * RPI * D * 2);
    }
  };
  auto issue_v = [&](int t) {
    const uint16_t *kp, *vp;
    int last;
    rows(t, wave * WR, kp, vp, last);
    vp = uniform_ptr(vp);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = i * RPI + lane / CH;
      const uint32_t rr = min(r, last);
      dma16(vp, 2 * (rr * static_cast<uint32_t>(vstride) + 8 * ((lane % CH) ^ swz_v<D>(wave * WR + r))),
            ldsw + (NS + (t - t0) % NS) * kTile + i * RPI * D * 2);
    }
  };

  const int l16 = lane & 15;
  // A operand of the second product: the wave's keys 16 s4 .. +16, elements 32 dt .. +32
  auto value_frag = [&](const char* vl, int s4, int dt) {
    const int r0 = key0 + 16 * s4 + 4 * hf + (l16 >> 2);
    const int c = 4 * dt + 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
    const u32x2 lo = read_tr(vl + r0 * D * 2 + 16 * (c ^ swz_v<D>(r0)) + 8 * (l16 & 1));
    const u32x2 hi = read_tr(vl + (r0 + 8) * D * 2 + 16 * (c ^ swz_v<D>(r0 + 8)) + 8 * (l16 & 1));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto scores32 = [&](const char* kl, int kt, f32x16& s) {
    s = f32x16{};
    const int row = key0 + 32 * kt + n;
    const char* kr = kl + row * D * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      s = mfma32(as_bf16x8(*reinterpret_cast<const u32x4*>(kr + 16 * ((2 * ks + hf) ^ swz_k<D>(row)))), q[ks], s);
  };
  auto scores = [&](const char* kl, f32x16 (&s)[KT]) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) scores32(kl, kt, s[kt]);
  };
  // the largest score of the lane's row, times c2
  auto top_of = [&](const f32x16 (&s)[KT]) {
    float top = fmaxf(s[0][0], s[KT - 1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(fmaxf(top, s[0][i]), s[KT - 1][i]);
    return max_across32(top) * c2;
  };
  // the reference point follows the maximum once it lags by more than 2^8: p stays
  // below 2^8, and most tiles leave o as it is
  auto follow = [&](float top) {
    if (__any(top > st.m + 8.0f)) {
      const float mn = fmaxf(st.m, top);
      const float f = st.m == mn ? 1.0f : __builtin_amdgcn_exp2f(st.m - mn);
      st.m = mn;
      st.l *= f;
      if constexpr (kExact) st.exact *= f;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) st.o[dt] *= f;
    }
  };
  auto weights = [&](const f32x16 (&s)[KT], bf16x8 (&p)[2 * KT]) {
    const float mu = st.m == kNegInf ? 0.0f : st.m;
    u32x4 w[2 * KT];
#pragma unroll
    for (int s4 = 0; s4 < 2 * KT; ++s4) {
      // p to bf16: at most 2^-8 of each, of random sign over the keys, next to the output's own
      // rounding of 2^-8.  As the sum of two bf16, with two products each, 8192 tokens of 32 heads of 128
      // take 695 instead of 488 us, 16 prompts of 5375 tokens together 37 instead of 25.5.
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float lo = __builtin_amdgcn_exp2f(s[s4 >> 1][8 * (s4 & 1) + 2 * i] * c2 - mu);
        const float hi = __builtin_amdgcn_exp2f(s[s4 >> 1][8 * (s4 & 1) + 2 * i + 1] * c2 - mu);
        if constexpr (kExact) st.exact += lo + hi;
        w[s4][i] = pack_bf16(lo, hi);
      }
      p[s4] = as_bf16x8(w[s4]);
    }
    // The sum is that of the rounded weights, which the product uses: a row whose visible values are all the
    // same gives that value.  8192 tokens of 32 heads take 470 -> 474 us for it, six prompts of 1500 of 16
    // 74.4 -> 76.4, shorter ones the same; the rounded weights added one by one 4.5 % more.
    float even = 0.0f, odd = 0.0f;
#pragma unroll
    for (int s4 = 0; s4 < 2 * KT; ++s4)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        even = add_bf16_pair(w[s4][i], even);
        odd = add_bf16_pair(w[s4][i + 1], odd);
      }
    st.l += even + odd;
  };
  auto values = [&](const char* vl, const bf16x8 (&p)[2 * KT]) {
#pragma unroll
    for (int s4 = 0; s4 < 2 * KT; ++s4)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) st.o[dt] = mfma32(as_bf16x8(value_frag(vl, s4, dt)), p[s4], st.o[dt]);
  };

  // A tile's scores are made while the weights of the tile before are: the matrix pipe
  // and the vector pipe have work of one wave at the same time.  Between two barriers, tile
  // t + 1's K and tile t's V are read; tile t + 2's K and tile t + 1's V are asked for, to be
  // there at the next (four buffers and loads two tiles earlier took the same time).
  int* flags = reinterpret_cast<int*>(lds + 2 * NS * kTile);   // of tiles j, by j mod 2
  if (threadIdx.x == 0) flags[0] = flags[1] = 0;
  issue_k(t0);
  issue_v(t0);
  if (t0 + 1 < t1) issue_k(t0 + 1);
  wait_barrier();
  // The order of issue: four fragments of K ahead, then behind every product the next
  // fragment and the vector work that its time covers (8192 tokens, 32 heads of 128: 492 us as the
  // compiler orders it, 484 with the products' order, 476 with the loads of K
  // behind the first products)
  // reads of V (two a fragment) in the place of those of K that are made already; of heads of 64 with
  // half the keys there are few products to hide them behind (2048 tokens 22.8 -> 21.5 us; whole tiles need the
  // registers for a third wave)
  constexpr int kAhead = D == 64 && KT == 1 ? 3 : 1;
  // vector instructions behind each of the first and of the second products (2048 tokens, 16 heads of 64: 23.8 us with 6 and
  // 10, 22.1 with 10 and 10; 8192, 32 of 128: 498 with 3 and 4, 502 with 4 and 4)
  constexpr int kFirst = D == 64 ? 10 : 3, kSecond = D == 64 ? 10 : 4;
  auto order = [&]() {
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < KT * KS - 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, kFirst, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, kFirst, 0);
    }
#pragma unroll
    for (int i = 0; i < KT * D / 16; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, kSecond, 0);
    }
  };
  f32x16 s[KT];
  scores(lds, s);
  float top = top_of(s);
  int j = 0;                                         // tile t0 + j
  {
    // tiles up to NS before the last that all rows of the workgroup see in full: the
    // lanes' offsets from a tile's first row stay the same.  K's chunks are placed by
    // the row in the tile, V's by its last bits, which are the same in every load
    uint32_t koff[NI], voff;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = i * RPI + lane / CH;
      koff[i] = 2 * (r * static_cast<uint32_t>(kstride) + 8 * ((lane % CH) ^ swz_k<D>(wave * WR + r)));
    }
    voff = 2 * (lane / CH * static_cast<uint32_t>(vstride) + 8 * ((lane % CH) ^ swz_v<D>(lane / CH)));
    const int full = min(t1, (b_min + 1) / kFlKeys) - NS - t0;   // tile t0 + full + NS - 1 is the last full one
    auto step = [&](const f32x16 (&s)[KT], f32x16 (&next)[KT]) {
      wait_barrier();
      const uint16_t *kp, *vp, *unused;
      int last;
      rows(t0 + j + NS, wave * WR, kp, unused, last);
      rows(t0 + j + NS - 1, wave * WR, unused, vp, last);
      kp = uniform_ptr(kp);
      vp = uniform_ptr(vp);
      const uint32_t kd = ldsw + (j % NS) * kTile, vd = ldsw + (NS + (j + NS - 1) % NS) * kTile;
      const char* kl = lds + ((j + 1) % NS) * kTile;
#pragma unroll
      for (int i = 0; i < NI; ++i) dma16(vp + i * RPI * vstride, voff, vd + i * RPI * D * 2);
      follow(top);
      bf16x8 p[2 * KT];
      scores(kl, next);
#pragma unroll
      for (int i = 0; i < NI; ++i) dma16(kp, koff[i], kd + i * RPI * D * 2);
      weights(s, p);
      values(lds + (NS + j % NS) * kTile, p);
      order();
      top = top_of(next);
      ++j;
    };
    // two at a time: the scores change places without moves
    f32x16 other[KT];
    for (; j + 1 < full;) {
      step(s, other);
      step(other, s);
    }
    if (j < full) {
      step(s, other);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[kt] = other[kt];
    }
  }
  // The last of them, and tiles that some rows see a part of, or nothing: there an
  // infinite or NaN value must not reach the rows that do not see it.
  auto ready = [&](int t) {                          // all of tile t's values are finite
    const bool edge = t * kFlKeys + kFlKeys - 1 > b_min;
    if (edge) {
      // what the wave itself has loaded, before the barrier that tells the others; the
      // flag of the tile after next is set behind the next barrier, when this one has been read
      wait_loads();
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(lds + (NS + j % NS) * kTile + wave * WR * D * 2 + i * 1024 + 16 * lane);
        bits |= nonfinite_bits(x[0]) | nonfinite_bits(x[1]) | nonfinite_bits(x[2]) | nonfinite_bits(x[3]);
      }
      if (bits) flags[j & 1] = 1;
    }
    wait_barrier();
    if (t + NS - 1 < t1) issue_v(t + NS - 1);
    if (t + NS < t1) issue_k(t + NS);
    return !edge || __builtin_amdgcn_readfirstlane(flags[j & 1]) == 0;
  };
  auto prepare = [&](int t, f32x16 (&s)[KT]) {
    const bool finite = ready(t);
    if (t * kFlKeys + kFlKeys - 1 > w_min) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t * kFlKeys + key0 + 32 * kt + 8 * (i >> 2) + 4 * hf + (i & 3) > lim) s[kt][i] = kNegInf;
      top = top_of(s);
    }
    follow(top);
    if (!finite) {
      // rarely: infinite and NaN values to the rows that see them, then out of the tile
      char* vl = lds + (NS + j % NS) * kTile;
#pragma unroll 1
      for (int key = key0; key < key0 + 32 * KT; ++key) {
        int row = key;
        asm volatile("" : "+v"(row));                // keeps the addresses out of registers
        const bool seen = t * kFlKeys + row <= lim;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(vl + row * D * 2 + 16 * ((4 * dt + g) ^ swz_v<D>(row)) + 8 * hf);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              st.o[dt][4 * g + i] += seen ? nonfinite_only(static_cast<uint16_t>(x[i >> 1] >> (16 * (i & 1)))) : 0.0f;
          }
      }
      wait_barrier();
#pragma unroll 1
      for (int i = threadIdx.x; i < kTile / 4; i += 64 * NW) {
        uint32_t* x = reinterpret_cast<uint32_t*>(vl + 4 * i);
        *x = finite_only(*x);
      }
      wait_barrier();
    }
  };
  for (; t0 + j + 1 < t1; ++j) {
    prepare(t0 + j, s);
    f32x16 next[KT];
    bf16x8 p[2 * KT];
    scores(lds + ((j + 1) % NS) * kTile, next);
    weights(s, p);
    values(lds + (NS + j % NS) * kTile, p);
    order();
    top = top_of(next);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) s[kt] = next[kt];
  }
  prepare(t0 + j, s);
  bf16x8 p[2 * KT];
  weights(s, p);
  values(lds + (NS + j % NS) * kTile, p);
}

// flash for keys and values in 8 bits of which every row sees the first n_keys (a prefix): four waves, 32 rows each.
// rows(tile, &k, &v, &k_scale, &v_scale) gives the wave's 16 rows of a tile, D codes each and one scale, and returns how many
// rows after the first may be read.  Codes come to registers a step ahead, and go to LDS as the bf16 that flash
// reads, so every wave converts a quarter of a tile once for all.  A NaN is seen by all rows, so nothing is kept
// from any.  Weights are one bf16 each in the second product, as in flash: as the sum of two, with two products each, 64 sequences
// behind 16385 keys take 41.1 us instead of 35.5, and their outputs are 0.00167 of their size from the definition in 64 bits
// instead of 0.00176 (outputs of float32 operations, rounded to bf16 once: 0.00167).
template <int D, bool kExact, class Rows>
__device__ __forceinline__ void flash_codes(const bf16x8 (&q)[D / 16], int t0, int t1, int n_keys, float c2, char* lds, Rows rows,
                                            FlashRows<D>& st) {
  t0 = __builtin_amdgcn_readfirstlane(t0);
  t1 = __builtin_amdgcn_readfirstlane(t1);
  if (t0 >= t1) return;
  constexpr int NW = 4, KS = D / 16, WR = kFlKeys / NW, CH = D / 16, RPI = 64 / CH, NI = WR / RPI, kTile = kFlKeys * D * 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hf = lane >> 5, l16 = lane & 15;
  struct Raw { u32x4 c[NI]; float scale; };
  Raw rk, rv;
  auto load = [&](int t, bool is_v, Raw& raw) {
    const uint8_t *kp, *vp;
    float ks, vs;
    const int last = rows(t, kp, vp, ks, vs);
    raw.scale = is_v ? vs : ks;
    const uint8_t* p = uniform_ptr(is_v ? vp : kp);
#pragma unroll
    for (int i = 0; i < NI; ++i) raw.c[i] = ldg16(p + min(i * RPI + lane / CH, last) * D + 16 * (lane % CH));
  };
  // to tile t's buffer, of K or V
  auto put = [&](int t, bool is_v, const Raw& raw) {
    char* tile = lds + ((is_v ? kFlBuffers : 0) + (t - t0) % kFlBuffers) * kTile;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = wave * WR + i * RPI + lane / CH, swz = is_v ? swz_v<D>(r) : swz_k<D>(r);
      u32x2 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = codes_to_bf16(raw.c[i][j], raw.scale);
      char* row = tile + r * D * 2;
      *reinterpret_cast<u32x4*>(row + 16 * ((2 * (lane % CH)) ^ swz)) = u32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
      *reinterpret_cast<u32x4*>(row + 16 * ((2 * (lane % CH) + 1) ^ swz)) = u32x4{w[2][0], w[2][1], w[3][0], w[3][1]};
    }
  };
  auto value_frag = [&](const char* vl, int s4, int dt) {
    const int r0 = 16 * s4 + 4 * hf + (l16 >> 2);
    const int c = 4 * dt + 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
    const u32x2 lo = read_tr(vl + r0 * D * 2 + 16 * (c ^ swz_v<D>(r0)) + 8 * (l16 & 1));
    const u32x2 hi = read_tr(vl + (r0 + 8) * D * 2 + 16 * (c ^ swz_v<D>(r0 + 8)) + 8 * (l16 & 1));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto scores = [&](int t, f32x16 (&s)[2]) {
    const char* kl = lds + (t - t0) % kFlBuffers * kTile;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = f32x16{};
      const int row = 32 * kt + n;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[kt] = mfma32(as_bf16x8(*reinterpret_cast<const u32x4*>(kl + row * D * 2 + 16 * ((2 * ks + hf) ^ swz_k<D>(row)))), q[ks], s[kt]);
    }
  };
  auto top_of = [&](const f32x16 (&s)[2]) {
    float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(fmaxf(top, s[0][i]), s[1][i]);
    return max_across32(top) * c2;
  };
  // as in flash
  auto attend = [&](int t, float top, const f32x16 (&s)[2]) {
    if (__any(top > st.m + 8.0f)) {
      const float mn = fmaxf(st.m, top);
      const float f = st.m == mn ? 1.0f : __builtin_amdgcn_exp2f(st.m - mn);
      st.m = mn;
      st.l *= f;
      if constexpr (kExact) st.exact *= f;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) st.o[dt] *= f;
    }
    const float mu = st.m == kNegInf ? 0.0f : st.m;
    const char* vl = lds + (kFlBuffers + (t - t0) % kFlBuffers) * kTile;
    float even = 0.0f, odd = 0.0f;
#pragma unroll
    for (int s4 = 0; s4 < 4; ++s4) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float lo = __builtin_amdgcn_exp2f(s[s4 >> 1][8 * (s4 & 1) + 2 * i] * c2 - mu);
        const float hi = __builtin_amdgcn_exp2f(s[s4 >> 1][8 * (s4 & 1) + 2 * i + 1] * c2 - mu);
        if constexpr (kExact) st.exact += lo + hi;
        w[i] = pack_bf16(lo, hi);
      }
      even = add_bf16_pair(w[0], even);
      odd = add_bf16_pair(w[1], odd);
      even = add_bf16_pair(w[2], even);
      odd = add_bf16_pair(w[3], odd);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) st.o[dt] = mfma32(as_bf16x8(value_frag(vl, s4, dt)), as_bf16x8(w), st.o[dt]);
    }
    st.l += even + odd;
  };
  // LDS writes are done, then the workgroup's barrier; loads to registers may be on their way
  auto barrier = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  load(t0, false, rk);
  load(t0, true, rv);
  put(t0, false, rk);
  put(t0, true, rv);
  if (t0 + 1 < t1) {
    load(t0 + 1, false, rk);
    load(t0 + 1, true, rv);
    put(t0 + 1, false, rk);
  }
  if (t0 + 2 < t1) load(t0 + 2, false, rk);
  barrier();
  // Between two barriers: tile t + 1's scores and tile t's values are read; K of t + 2 and V of t + 1, which have come to
  // registers, are put where those of t and t - 1 were, and the next are asked for.
  f32x16 s[2];
  scores(t0, s);
  float top = top_of(s);
  for (int t = t0; t + 1 < t1; ++t) {
    barrier();                       // K of t has been read, V of t - 1 too
    f32x16 next[2];
    scores(t + 1, next);
    attend(t, top, s);
    put(t + 1, true, rv);
    if (t + 2 < t1) {
      put(t + 2, false, rk);
      load(t + 2, true, rv);
      if (t + 3 < t1) load(t + 3, false, rk);
    }
    top = top_of(next);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) s[kt] = next[kt];
  }
  barrier();
  const int last = t1 - 1;
  if (last * kFlKeys + kFlKeys > n_keys) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (last * kFlKeys + 32 * kt + 8 * (i >> 2) + 4 * hf + (i & 3) >= n_keys) s[kt][i] = kNegInf;
    top = top_of(s);
  }
  attend(last, top, s);
}

// The two waves of 32 rows (KH 2) put their keys together: afterwards both have the
// rows' maximum and their parts of the sums; of o, in registers o[0 .. D / 64), the wave of half 0 has
// elements 0 .. D / 2 and that of half 1 the others.  For all NW waves.
template <int D, int NW>
__device__ __forceinline__ void add_halves(FlashRows<D>& st, char* lds) {
  constexpr int DT = D / 64, kWave = 64 * (16 * DT + 2) * 4;
  static_assert(NW * kWave <= flash_lds<D>(), "in the tiles' LDS");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool up = wave >= NW / 2;
  char *mine = lds + wave * kWave + 16 * lane, *other = lds + (wave ^ (NW / 2)) * kWave + 16 * lane;
  __syncthreads();                                   // the last tile's reads are done
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const f32x16 give = up ? st.o[dt] : st.o[DT + dt];
    if (up) st.o[dt] = st.o[DT + dt];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<f32x4*>(mine + (4 * dt + c) * 1024) = f32x4{give[4 * c], give[4 * c + 1], give[4 * c + 2], give[4 * c + 3]};
  }
  *reinterpret_cast<float2*>(mine + DT * 4096 - 8 * lane) = float2{st.m, st.l};
  __syncthreads();
  const float2 ml = *reinterpret_cast<const float2*>(other + DT * 4096 - 8 * lane);
  const float top = fmaxf(st.m, ml.x), mu = top == kNegInf ? 0.0f : top;
  const float f = __builtin_amdgcn_exp2f(st.m - mu), fo = __builtin_amdgcn_exp2f(ml.x - mu);
  st.m = top;
  st.l = st.l * f + ml.y * fo;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(other + (4 * dt + c) * 1024);
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[dt][4 * c + i] = st.o[dt][4 * c + i] * f + x[i] * fo;
    }
}

}  // namespace dsk
