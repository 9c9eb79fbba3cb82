// Attention of a decode or verify step over the paged cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e)
//
// The M = q_len * heads / kv_heads query rows that share a key head are the
// columns of 16-wide MFMA tiles; each 32 keys of a wave cost 2 D/32 products
// for K q^T and 2 D/16 for V^T p^T (p as two bf16) and 4 D bytes of cache per key, so the
// stream of the cache bounds the kernel and everything else has to stay out of its
// way: K and V go straight into registers (no LDS, no barrier in the loop).
//
// S^T = K q^T comes out with a query row in every lane (column lane & 15) and
// keys 4g + r of a 16-key tile in lane group g = lane >> 4.  That is a B
// operand of the second product already: the contraction may run over the keys
// in any order, so slots 0..3 of group g are given keys 4g..4g+3 of the first
// tile and slots 4..7 those of the second, and p never crosses lanes.  V^T as
// the A operand then wants, in lane (m, g), those eight keys at one element
// d(m, t) per product t.  The lane loads VW = D / 16 consecutive elements
// VW m.. of each of its keys (whole 16-byte pieces) and picks element t of all
// eight with byte permutes: d(m, t) = VW m + t.  Column q of O^T stays in lane
// q, so the running maximum and the rescaling are lane-local too.
//
// Work: the (sequence, key head) items' 128-key units in a row, cut into equal
// shares for a fixed number of workgroups, so ragged lengths cost no balance
// and the lengths are read on the device (a captured launch follows them).  An
// item that lies in one share is finished there; the parts of the others go
// through float32 partial rows (o, m, l) and k_paged_join.  Short tables
// need neither: a workgroup of eight waves takes a whole item.
//
// 64 sequences of 1 to 8192 keys, 32 + 8 heads of 128: 74 us for 381 MB of cache (5.1 TB/s, as
// a large copy) and 5 us for the join.  8 of up to 32768, 16 + 4 heads of 64, two tokens: 15 us
// for 66 MB and 5 us: 512 workgroups of few loads each, so the start (lengths, pages,
// keys, one after the other) and the join count.
//
// A prefix that the batch shares is a pass of its own over all of the batch's rows
// (flash, attn_core.h), split along its keys; its workgroups come first in the
// launch of the shares, so that its products run beside their loads (a launch of its own: 51 against 41 us
// for 16385 keys and 64 sequences).  There the kernel takes 29 us: 9 us from the launch to the
// first tile's end and for 16.8 MB of partial rows, 1 us for each of 16 tiles, the rest the
// shares' loads beside them; the join of 16 parts and the own keys' takes 6.6 us.
//
// A cache in 8 bits (kv8.h) is the same kernel with codes made to bf16 in registers, exactly.  64 sequences of 1
// to 8192 keys: 26 us for 101 MB, of which the bytes are 17 at the 6 TB/s that long sequences reach, a workgroup's start and
// end most of the rest, and 4.8 us for the join.  The prefix of 16385 keys: 33 us beside 29 in bf16, since its products,
// not its bytes, bound it and the conversions come to them.
//
// Weights of the keys need every row's final sum, so scores wait in float32 for a pass of their own beside (or behind) the
// join: 8 M bytes a key and head more, against 4 D (2 D) for the key and value.  With few rows that is little: 48
// sequences of up to 2100 keys, four rows, 16 us and 5.8 for the join and weights; with 64 rows the weights take as long as all else.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "attn_core.h"

namespace dsk {
namespace {

constexpr int kPgThreads = 256;
// Keys of a wave's step, in tiles of 16.  Also of codes, which are half the bytes: with 64 their conversions spill (64
// sequences of up to 8192 keys of 128 37.8 us, 29.9 with 32; 8 of up to 32768 keys of 64 21.2 and 19.4).
constexpr int kPgStep = 32, kPgTiles = kPgStep / 16;
constexpr int kPgUnit = 4 * kPgStep; // of which shares are made: a step of each of four waves
// Units that an item counts for beside its keys'.  It has a start and an end of its own, about 4 us, beside which codes are
// little: 64 sequences of 1 to 8192 keys of 128 take 29.9 us with 1, 30.4 with 2, 33.6 with 4 (and with steps of 64
// keys 37.8 with 1, 52.8 with none); 8 of up to 32768 of 64 19.4, 18.8, 18.7.
template <bool F8>
constexpr uint32_t item_units() { return F8 ? 1 : 0; }
constexpr int kPgShort = 512;       // keys of a table row that one workgroup takes alone
constexpr int kPgShortMany = 1024;  // where there are kPgMany items, or codes to read
constexpr int kPgMany = 512;
constexpr int kPgShortWaves = 8;
constexpr int64_t kPgFewKeys = 512 << 10;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct PagedArgs {
  const uint16_t* q;
  uint16_t* out;
  const int32_t* lens;
  CacheView c;
  float* po;                        // partial rows [slot][M][D]
  float* pml;                       // [slot][M][2]: maximum (of scores times c), sum
  i32x2* parts;                     // of an item with keys: its first slot, and how many parts to join
  float* pre_o;                     // prefix partials [split][kv head][batch * M][D]
  float* pre_ml;
  const int32_t* pages;             // of the prefix
  int64_t q_token, q_head, o_token, o_head;
  float c2;                         // scale * log2(e)
  int32_t batch, q_len, kv_heads, group, prefix, shares, splits;
  int32_t row_tiles, prefix_blocks; // of the prefix: tiles of all rows, workgroups
  const uint8_t *k_scale, *v_scale; // of a cache in 8 bits
  float* weights;                   // of the cache's rows, to be added to, or null; then also:
  float* scores;                    // [item][key of the table row][M rounded up to fours], times c
  float* lse;                       // [item][M]: log2 of the sum of 2^score (infinite: the row sees no key)
  float* pre_l;                     // the prefix partials' sums of the weights before their rounding to bf16
};

// Keys of sequence b that the cache can hold; `bad` if lens[b] claims more.
__device__ __forceinline__ int length_of(const PagedArgs& a, int b, bool& bad) {
  const int n = a.lens[b], cap = a.c.max_pages << a.c.page_shift;
  bad = n > cap;
  return min(max(n, 0), cap);
}
template <bool F8>
__device__ __forceinline__ uint32_t units_of(int len) {
  return len > 0 ? (len + kPgUnit - 1) / kPgUnit + item_units<F8>() : 0;
}

template <int V>
struct Const { static constexpr int value = V; };

// Sums over the lanes 0 .. lane, in six vector additions.
__device__ __forceinline__ uint32_t sum_up_to_lane(uint32_t v) {
  auto add = [&](auto ctrl, auto rows) {
    v += __builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl.value, rows.value, 0xf, false);
  };
  add(Const<0x111>{}, Const<0xf>{});                 // the lane 1, 2, 4, 8 below, in rows of 16
  add(Const<0x112>{}, Const<0xf>{});
  add(Const<0x114>{}, Const<0xf>{});
  add(Const<0x118>{}, Const<0xf>{});
  add(Const<0x142>{}, Const<0xa>{});                 // lane 15 of the row below to rows 1 and 3
  add(Const<0x143>{}, Const<0xc>{});                 // lane 31 to rows 2 and 3
  return v;
}

// Units of one key head, 64 sequences at a time: lane's own, and up to its own.
// Fewer than 2^31 in all, times the key heads too.
struct Units { uint32_t own, up_to; };
template <bool F8>
__device__ __forceinline__ Units units_at(const PagedArgs& a, int b0) {
  const int b = b0 + (threadIdx.x & 63);
  bool bad;
  const uint32_t n = b < a.batch ? units_of<F8>(length_of(a, b, bad)) : 0;
  return Units{n, sum_up_to_lane(n)};
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

// LDS writes of a wave's lanes before the reads of others of its lanes.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int D, bool F8>
struct Step {                       // one wave's keys, in tiles of 16
  static constexpr int kPieces = D / (F8 ? 64 : 32);
  u32x4 k[kPgTiles][kPieces];
  uint32_t v[4 * kPgTiles][kPieces]; // VW = D / 16 elements of 4 keys of each
};

template <int N>
__device__ __forceinline__ void load_v(uint32_t (&v)[N], const void* p) {
  if constexpr (N == 4) {
    const u32x4 r = ldg16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r[i];
  } else if constexpr (N == 2) {
    const u32x2 r = ldg<u32x2>(p);
    v[0] = r[0];
    v[1] = r[1];
  } else {
    v[0] = ldg<uint32_t>(p);
  }
}

// bf16 values of four keys a tile, element t of each: slots 0..3 (4..7) of a product's A operand from tile 0 (1).
// Codes: four elements of four keys are a 4 x 4 of bytes; bytes of one element together, then to bf16.
template <int VW>
__device__ __forceinline__ void values_of(const uint32_t (&v)[4][VW / 4], float scale, u32x2 (&w)[VW]) {
#pragma unroll
  for (int i = 0; i < VW / 4; ++i)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const uint32_t sel = hi ? 0x07030602u : 0x05010400u;
      const uint32_t a = __builtin_amdgcn_perm(v[1][i], v[0][i], sel), b = __builtin_amdgcn_perm(v[3][i], v[2][i], sel);
      w[4 * i + 2 * hi] = codes_to_bf16(__builtin_amdgcn_perm(b, a, 0x05040100u), scale);
      w[4 * i + 2 * hi + 1] = codes_to_bf16(__builtin_amdgcn_perm(b, a, 0x07060302u), scale);
    }
}

// LDS of a segment of W waves: their rows, then maxima and sums.
template <int D, int RT, int W>
struct SegLds {
  float o[W][16][D + 4];
  float ml[W][16 * RT][2];
};

// Lane 2 i + kt: the page of the wave's 16-key tile kt in step kk + i of those that begin at
// tile `tile0` (the table row's last one behind its end; the sequence's length need not be known yet).
template <int W>
__device__ __forceinline__ int page_ids(const PagedArgs& a, int b, int tile0, int kk) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tile = tile0 + (static_cast<int64_t>(kk) + (lane >> 1)) * (2 * W) + 2 * wave + (lane & 1);
  const int page = static_cast<int>(min(tile >> (a.c.page_shift - 4), static_cast<int64_t>(a.c.max_pages - 1)));
  return ldg<int32_t>(a.c.table + b * a.c.table_stride + page);
}

// Keys [start, stop) of item (b, h), whole steps of a wave, for the rows from
// r0 on: to `out` (slot < 0: they are all of the item's) or to the partial rows of `slot`.
// first_ids: page_ids of start.
//
// F8: a cache in 8 bits.  A lane's piece of a key is D / 4 codes, of which product ks takes 8 (queries
// are held in the same order), so that K too comes in 16-byte loads; a 16-key tile is a block of one scale, which the
// conversion to bf16 applies.  kWeigh: scores are kept for k_key_weights.
template <int D, int RT, int W, bool F8, bool kWeigh>
__device__ __forceinline__ void segment(const PagedArgs& a, int b, int h, int len, bool bad_len, int r0, int start, int stop,
                                        int64_t slot, int first_ids, SegLds<D, RT, W>& lds) {
  using S = Step<D, F8>;
  constexpr int VW = D / 16, KS = D / 32, kUnit = kPgStep * W;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  const int M = a.q_len * a.group;
    // queries: column n16 of row tile rt is row 16 rt + n16 = token * group + head of the group
    bf16x8 q[RT][KS];
    int lim[RT];                    // last key that the lane's row sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = min(r0 + 16 * rt + n16, M - 1), tok = r / a.group, hd = h * a.group + r % a.group;
      const uint16_t* p = a.q + (static_cast<int64_t>(b) * a.q_len + tok) * a.q_token + hd * a.q_head + (F8 ? D / 4 : 8) * g;
      lim[rt] = len - a.q_len + tok;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) q[rt][ks] = as_bf16x8(ldg16(p + (F8 ? 8 : 32) * ks));
    }
    f32x4 o[RT][VW];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = kNegInf;
      l[rt] = bad_len ? __builtin_nanf("") : 0.0f;
#pragma unroll
      for (int t = 0; t < VW; ++t) o[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const int32_t* trow = a.c.table + b * a.c.table_stride;
    const int last_tile = (len - 1) >> 4, first_tile = start >> 4;
    stop = min(stop, len);
    const int k1 = (stop - start + kUnit - 1) / kUnit;   // steps of W waves
    int ids = first_ids, ids0 = 0;    // lane 2 i + kt: the page of tile kt of step ids0 + i
    int bad_tile = INT32_MAX;         // the lane's first 16 keys on a page outside the cache
    // F8: scale bytes of the lane's tile, and those of the ids before, which a step may still need
    uint32_t k_byte = 0, v_byte = 0, old_k_byte = 0, old_v_byte = 0;
    int old0 = 0;
    auto check_ids = [&]() {
      const int tile = first_tile + (ids0 + (lane >> 1)) * (2 * W) + 2 * wave + (lane & 1);
      const bool out_of = ids < 0 || ids >= a.c.n_pages;
      if (out_of && tile * 16 < stop) bad_tile = min(bad_tile, tile);
      if (out_of) ids = 0;
      if constexpr (F8) {
        const int64_t at = ((static_cast<int64_t>(ids) * a.kv_heads + h) << (a.c.page_shift - 4)) +
                           (tile & ((1 << (a.c.page_shift - 4)) - 1));
        old_k_byte = k_byte;
        old_v_byte = v_byte;
        k_byte = ldg<uint8_t>(a.k_scale + at);
        v_byte = ldg<uint8_t>(a.v_scale + at);
      }
    };
    check_ids();
    auto load = [&](S& s, int kk) {
      if (kk - ids0 >= 32) {
        old0 = ids0;
        ids0 = kk;
        ids = page_ids<W>(a, b, first_tile, kk);
        check_ids();
      }
      const int tile0 = first_tile + kk * (2 * W) + 2 * wave;
      if (tile0 * 16 >= stop) return;                 // none of the wave's keys in this step
#pragma unroll
      for (int kt = 0; kt < kPgTiles; ++kt) {
        const int tile = min(tile0 + kt, last_tile);
        const int id = __builtin_amdgcn_readlane(ids, 2 * (kk - ids0) + tile - tile0);
        const int last_row = len - 1 - tile * 16;     // rows past the length: the last one again
        const int row0 = (tile * 16) & ((1 << a.c.page_shift) - 1);
        const int64_t base = (((static_cast<int64_t>(id) * a.kv_heads + h) << a.c.page_shift) + row0) * D;
        if constexpr (F8) {
          const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.c.k) + base + min(n16, last_row) * D + D / 4 * g;
#pragma unroll
          for (int i = 0; i < S::kPieces; ++i) s.k[kt][i] = ldg16(kp + 16 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            load_v(s.v[4 * kt + j], reinterpret_cast<const uint8_t*>(a.c.v) + base + min(4 * g + j, last_row) * D + VW * n16);
        } else {
          const uint16_t* kp = a.c.k + base + min(n16, last_row) * D + 8 * g;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) s.k[kt][ks] = ldg16(kp + 32 * ks);
#pragma unroll
          for (int j = 0; j < 4; ++j) load_v(s.v[4 * kt + j], a.c.v + base + min(4 * g + j, last_row) * D + VW * n16);
        }
      }
    };
    // rarely: infinite and NaN values of step kk, to the rows that see them (the
    // products then leave them out)
    auto add_nonfinite = [&](int kk) {
#pragma unroll 1
      for (int key = start + kk * kUnit + kPgStep * wave, end = min(key + kPgStep, len); key < end; ++key) {
        int id = ldg<int32_t>(trow + (key >> a.c.page_shift));
        if (id < 0 || id >= a.c.n_pages) id = 0;
        const int in_page = key & ((1 << a.c.page_shift) - 1);
        const int64_t row = ((static_cast<int64_t>(id) * a.kv_heads + h) << a.c.page_shift) + in_page;
        const bool no_scale = F8 && ldg<uint8_t>(a.v_scale + (F8 ? row / kScaleRows : 0)) > kMostScale;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int t = 0; t < VW; ++t) {
            float x;
            if constexpr (F8) {
              const uint32_t c = ldg<uint8_t>(reinterpret_cast<const uint8_t*>(a.c.v) + row * D + VW * (4 * g + r) + t);
              x = no_scale || (c & 0x7fu) == 0x7fu ? __builtin_nanf("") : 0.0f;
            } else {
              x = nonfinite_only(ldg<uint16_t>(a.c.v + row * D + VW * (4 * g + r) + t));
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][t][r] += key <= lim[rt] ? x : 0.0f;
          }
      }
    };
    auto compute = [&](const S& s, int kk) {
      const int key0 = start + kk * kUnit + kPgStep * wave;
      if (key0 >= stop) return;
      const bool masked = key0 + kPgStep - 1 > len - a.q_len;
      float k_scale[kPgTiles], v_scale[kPgTiles];
      bool good_scales = true;
      if constexpr (F8) {
        const bool old = kk < ids0;
        const uint32_t kb = old ? old_k_byte : k_byte, vb = old ? old_v_byte : v_byte;
        const int tile0 = key0 >> 4;
#pragma unroll
        for (int kt = 0; kt < kPgTiles; ++kt) {
          const int at = 2 * (kk - (old ? old0 : ids0)) + min(tile0 + kt, last_tile) - tile0;
          k_scale[kt] = scale_of(lane_value(kb, at));
          const uint32_t byte = lane_value(vb, at);
          good_scales = good_scales && byte <= kMostScale;
          v_scale[kt] = scale_of(byte);
        }
      }
      // An infinite value times a weight's rest, which may be zero or negative, or the weight zero of a key that a
      // row does not see or of a place behind the last key (that key's values again), would be NaN: are
      // all the values finite?  The largest exponents of the pairs tell (decode_64 0.5 us more than without).
      // Codes have no infinity, and a NaN that every row sees may go through the products: there the question is
      // for the last keys alone.
      auto all_finite = [&]() {
        if constexpr (F8) {
          if (!masked) return true;
          uint32_t bits = 0;
#pragma unroll
          for (int j = 0; j < 4 * kPgTiles; ++j)
#pragma unroll
            for (int i = 0; i < S::kPieces; ++i) bits |= nan_codes(s.v[j][i]);
          return good_scales && !__any(bits != 0);
        } else {
          u16x2 largest = {0, 0};
#pragma unroll
          for (int j = 0; j < 4 * kPgTiles; ++j)
#pragma unroll
            for (int i = 0; i < VW / 2; ++i)
              largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16x2, s.v[j][i] & 0x7f807f80u));
          return !__any(nonfinite_bits(__builtin_bit_cast(uint32_t, largest)) != 0);
        }
      };
      bf16x8 p[RT], rest[RT];       // the weights: bf16, and what that rounds off
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 x[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          x[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            u32x4 key;
            if constexpr (F8) {
              const u32x4 c = s.k[kt][ks / 2];
              const u32x2 lo = codes_to_bf16(c[2 * (ks & 1)], k_scale[kt]), hi = codes_to_bf16(c[2 * (ks & 1) + 1], k_scale[kt]);
              key = u32x4{lo[0], lo[1], hi[0], hi[1]};
            } else {
              key = s.k[kt][ks];
            }
            x[kt] = mfma16(as_bf16x8(key), q[rt][ks], x[kt]);
          }
        }
        if (masked) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (key0 + 16 * kt + 4 * g + r > lim[rt]) x[kt][r] = kNegInf;
        }
        if constexpr (kWeigh) {
          const int row = r0 + 16 * rt + n16;
          const int64_t item = static_cast<int64_t>(b) * a.kv_heads + h;
          const int at = key0 + 4 * g;
          const int stride = (M + 3) & ~3;
          float* to = a.scores + (item * (static_cast<int64_t>(a.c.max_pages) << a.c.page_shift) + at) * stride + row;
          if (row < M)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (at + 16 * kt + r < len) to[(16 * kt + r) * stride] = x[kt][r] * a.c2;
        }
        float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                          fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
        top = max_across32(max_across16(top)) * a.c2;
        // the reference point follows the maximum once it lags by more than 2^8
        if (__any(top > m[rt] + 8.0f)) {
          const float mn = fmaxf(m[rt], top);
          const float f = m[rt] == mn ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mn);
          m[rt] = mn;
          l[rt] *= f;
#pragma unroll
          for (int t = 0; t < VW; ++t) o[rt][t] *= f;
        }
        const float mu = m[rt] == kNegInf ? 0.0f : m[rt];
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = __builtin_amdgcn_exp2f(x[i >> 2][i & 3] * a.c2 - mu);
          l[rt] += e[i];
        }
        // as the sum of two bf16: 2^-16 of each is left, far below the output's own rounding of 2^-8
        u32x4 w, u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = pack_bf16(e[2 * i], e[2 * i + 1]);
          u[i] = pack_bf16(e[2 * i] - __uint_as_float(w[i] << 16), e[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u));
        }
        p[rt] = as_bf16x8(w);
        rest[rt] = as_bf16x8(u);
      }
      const bool finite = all_finite();
      if (!finite) add_nonfinite(kk);
      u32x2 w0[VW], w1[VW];
      if constexpr (F8) {
        values_of<VW>(*reinterpret_cast<const uint32_t(*)[4][VW / 4]>(&s.v[0]), v_scale[0], w0);
        values_of<VW>(*reinterpret_cast<const uint32_t(*)[4][VW / 4]>(&s.v[4]), v_scale[1], w1);
      }
#pragma unroll
      for (int t = 0; t < VW; ++t) {
        u32x4 w;
        if constexpr (F8) {
          w = u32x4{w0[t][0], w0[t][1], w1[t][0], w1[t][1]};
        } else {
          const uint32_t sel = t & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(s.v[2 * i + 1][t / 2], s.v[2 * i][t / 2], sel);
        }
        if (!finite)
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = finite_only(w[i]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][t] = mfma16(as_bf16x8(w), rest[rt], mfma16(as_bf16x8(w), p[rt], o[rt][t]));
      }
    };

    S s0, s1;
    load(s0, 0);
    int kk = 0;
    for (; kk + 1 < k1; kk += 2) {
      load(s1, kk + 1);
      compute(s0, kk);
      if (kk + 2 < k1) load(s0, kk + 2);
      compute(s1, kk + 1);
    }
    if (kk < k1) compute(s0, kk);

    // the waves' parts
    const bool any_bad = __any(bad_tile != INT32_MAX);
    if (any_bad)
#pragma unroll
      for (int s = 32; s >= 1; s >>= 1) bad_tile = min(bad_tile, __shfl_xor(bad_tile, s, 64));
    __syncthreads();                 // the last segment's reads of LDS are done
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] = sum_across32(sum_across16(l[rt]));
      if (any_bad && (lim[rt] >> 4) >= bad_tile) l[rt] = __builtin_nanf("");   // the rows that see such keys
      if (g == 0) {
        lds.ml[wave][16 * rt + n16][0] = m[rt];
        lds.ml[wave][16 * rt + n16][1] = l[rt];
      }
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (rt) __syncthreads();
      float top = lds.ml[0][16 * rt + n16][0];
#pragma unroll
      for (int w = 1; w < W; ++w) top = fmaxf(top, lds.ml[w][16 * rt + n16][0]);
      const float f = top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m[rt] - top);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < VW; t += 4)
          *reinterpret_cast<f32x4*>(&lds.o[wave][n16][VW * (4 * g + r) + t]) =
              f32x4{o[rt][t][r], o[rt][t + 1][r], o[rt][t + 2][r], o[rt][t + 3][r]} * f;
      __syncthreads();
      const int row = threadIdx.x / (D / 8), d0 = 8 * (threadIdx.x % (D / 8));
      const int r = r0 + 16 * rt + row, rl = 16 * rt + row;
      if (row < 16 && r < M) {
        float mm = lds.ml[0][rl][0], ll = 0.0f;
#pragma unroll
        for (int w = 1; w < W; ++w) mm = fmaxf(mm, lds.ml[w][rl][0]);
        const float mu = mm == kNegInf ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < W; ++w) ll += lds.ml[w][rl][1] * __builtin_amdgcn_exp2f(lds.ml[w][rl][0] - mu);
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = lds.o[0][row][d0 + i];
#pragma unroll
          for (int w = 1; w < W; ++w) y[i] += lds.o[w][row][d0 + i];
        }
        if (slot < 0) {
          const int tok = r / a.group, hd = h * a.group + r % a.group;
          const bool sees = len - a.q_len + tok >= 0 || ll != ll;   // else no key: zeros
          const float inv = 1.0f / ll;
          if constexpr (kWeigh)
            if (d0 == 0) a.lse[(static_cast<int64_t>(b) * a.kv_heads + h) * M + r] = sees ? mm + log2f(ll) : -kNegInf;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = sees ? y[i] * inv : 0.0f;
          *reinterpret_cast<u32x4*>(a.out + (static_cast<int64_t>(b) * a.q_len + tok) * a.o_token + hd * a.o_head + d0) =
              u32x4{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7])};
        } else {
          float* po = a.po + (slot * M + r) * D + d0;
          *reinterpret_cast<f32x4*>(po) = f32x4{y[0], y[1], y[2], y[3]};
          *reinterpret_cast<f32x4*>(po + 4) = f32x4{y[4], y[5], y[6], y[7]};
          if (d0 == 0) *reinterpret_cast<float2*>(a.pml + (slot * M + r) * 2) = float2{mm, ll};
        }
      }
    }
}

// Workgroup `share` of a.shares takes its share of all units.
template <int D, int RT, bool F8, bool kWeigh>
__device__ __forceinline__ void shares(const PagedArgs& a, int share, int r0, SegLds<D, RT, 4>& lds) {
  constexpr uint32_t kHead = item_units<F8>();
  Units n;
  uint32_t all = 0;                  // units of one key head
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    n = units_at<F8>(a, b0);
    all += lane_value(n.up_to, 63);
  }
  const uint32_t total = all * a.kv_heads, quota = (total + a.shares - 1) / a.shares;
  uint32_t u0, u1;
  // in 8 bits shares that differ by one unit at most, of two units at least
  const uint32_t n_shares = F8 ? max(min(total / 2, static_cast<uint32_t>(a.shares)), min(total, 1u)) : a.shares;
  if constexpr (F8) {
    if (static_cast<uint32_t>(share) >= n_shares) return;
    const uint32_t each = total / n_shares, rest = total % n_shares;   // rest * share: below 2^18
    u0 = share * each + share * rest / n_shares;
    u1 = (share + 1) * each + (share + 1) * rest / n_shares;
  } else {
    u0 = share * quota;
    u1 = min(u0 + quota, total);
    if (u0 >= u1) return;
  }
  // the share that a unit lies in
  auto share_of = [&](uint32_t u) {
    if constexpr (F8) return static_cast<int>((static_cast<double>(u + 1) * n_shares - 1.0) / static_cast<double>(total));
    else return static_cast<int>(u / quota);
  };
  // the sequence that u0 lies in, and the units of one key head in those before it
  const uint32_t first_unit = u0 / a.kv_heads;
  uint32_t before = 0;
  int b = a.batch;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) n = units_at<F8>(a, b0);
    const uint64_t past = __ballot(before + n.up_to > first_unit);
    if (past) {
      const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
      before += lane_value(n.up_to - n.own, l);
      b = b0 + l;
      break;
    }
    before += lane_value(n.up_to, 63);
  }
  for (uint32_t u = u0; u < u1 && b < a.batch;) {
    bool bad_len;
    const int len = length_of(a, b, bad_len);
    const uint32_t nb = units_of<F8>(len), first = before * a.kv_heads;
    if (nb == 0 || u >= first + nb * a.kv_heads) {
      before += nb;
      ++b;
      continue;
    }
    // an item's first unit is kv_heads * before + h * its units
    const int h = static_cast<int>((u - first) / nb);
    const uint32_t item0 = first + h * nb, begin = u, end = min(item0 + nb, u1);
    u = end;
    const int k0 = static_cast<int>(max(begin, item0 + kHead) - item0 - kHead), k1 = static_cast<int>(end - item0) - static_cast<int>(kHead);
    if (k0 >= k1) continue;          // none of its keys: the next share begins with them
    const bool whole = k0 == 0 && end == item0 + nb;
    const int64_t slot = whole ? (a.splits ? 2 * static_cast<int64_t>(a.shares) + static_cast<int64_t>(b) * a.kv_heads + h : -1)
                               : 2 * static_cast<int64_t>(share) + (begin == u0 ? 0 : 1);
    if (k0 == 0 && r0 == 0 && threadIdx.x == 0)
      a.parts[b * a.kv_heads + h] =
          i32x2{static_cast<int>(slot), whole ? (a.splits ? 1 : 0) : share_of(item0 + nb - 1) - share + 1};
    segment<D, RT, 4, F8, kWeigh>(a, b, h, len, bad_len, r0, k0 * kPgUnit, k1 * kPgUnit, slot, page_ids<4>(a, b, k0 * (kPgUnit / 16), 0), lds);
  }
}

// All rows of the batch against a part of the prefix: tile `row_tile` of 128 rows of
// head h, split `split` of the keys.
constexpr int kPreWaves = 4;
constexpr int kPreRows = 32 * kPreWaves;
constexpr int kPreBlocks = 256;      // workgroups of the prefix, at most about: one a CU (prefix of 16385 keys for 64
                                     // sequences: 40 us, 45 with 128, 47 with 384, 50 with 512)
constexpr int kPreChunk = 64;        // tiles whose places in the cache a wave holds at once

template <int D, bool F8, bool kWeigh>
__device__ __forceinline__ void prefix_part(const PagedArgs& a, int block, char* lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hf = lane >> 5;
  const int h = block % a.kv_heads, rest = block / a.kv_heads, split = rest / a.row_tiles;
  const int rows = a.batch * a.q_len * a.group;      // at most 2^23
  const int wr0 = rest % a.row_tiles * kPreRows + 32 * wave;
  const int tiles = (a.prefix + kFlKeys - 1) / kFlKeys;
  const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits);
  const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);
  bf16x8 q[D / 16];
  const int rq = min(wr0 + n, rows - 1), tok = rq / a.group, hd = h * a.group + rq % a.group;
  const uint16_t* qp = a.q + tok * a.q_token + hd * a.q_head + 8 * hf;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) q[ks] = as_bf16x8(ldg16(qp + 16 * ks));
  FlashRows<D> st;
  st.m = kNegInf;
  st.l = st.exact = 0.0f;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) st.o[dt] = f32x16{};
  uint64_t bad = 0;
  // where the wave's rows of kPreChunk tiles lie in the cache, a tile a lane: flash's loop
  // has neither a branch nor a multiplication for them
  for (int c0 = t0; c0 < t1; c0 += kPreChunk) {
    const int c1 = min(c0 + kPreChunk, t1), row = wave * (kFlKeys / kPreWaves);
    const int key = min((c0 + lane) * kFlKeys + row, a.prefix - 1);
    int id = ldg<int32_t>(a.pages + (key >> a.c.page_shift));
    const bool out_of = id < 0 || id >= a.c.n_pages;
    bad |= __ballot(out_of && c0 + lane < c1);
    if (out_of) id = 0;
    const int64_t at = (((static_cast<int64_t>(id) * a.kv_heads + h) << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1))) * D;
    const int at_lo = static_cast<int>(at), at_hi = static_cast<int>(at >> 32);
    auto base_of = [&](int t) {
      const uint32_t lo = __builtin_amdgcn_readlane(at_lo, t - c0), hi = __builtin_amdgcn_readlane(at_hi, t - c0);
      return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
    };
    if (c0 > t0) __syncthreads();      // the last chunk's reads of LDS are done
    if constexpr (F8) {
      // a wave's 16 rows of a tile are a block of one scale
      const int k_byte = ldg<uint8_t>(a.k_scale + at / (kScaleRows * D)), v_byte = ldg<uint8_t>(a.v_scale + at / (kScaleRows * D));
      auto src = [&](int t, const uint8_t*& kp, const uint8_t*& vp, float& ks, float& vs) {
        const int64_t base = base_of(t);
        kp = reinterpret_cast<const uint8_t*>(a.c.k) + base;
        vp = reinterpret_cast<const uint8_t*>(a.c.v) + base;
        ks = scale_of(static_cast<uint32_t>(__builtin_amdgcn_readlane(k_byte, t - c0)));
        vs = scale_of(static_cast<uint32_t>(__builtin_amdgcn_readlane(v_byte, t - c0)));
        return max(a.prefix - 1 - (t * kFlKeys + row), 0);
      };
      flash_codes<D, kWeigh>(q, c0, c1, a.prefix, a.c2, lds, src, st);
    } else {
      auto src = [&](int t, int row, const uint16_t*& kp, const uint16_t*& vp, int& last) {
        const int64_t base = base_of(t);
        kp = a.c.k + base;
        vp = a.c.v + base;
        last = max(a.prefix - 1 - (t * kFlKeys + row), 0);
      };
      flash<D, kPreWaves, 1, kWeigh>(q, c0, c1, a.prefix - 1, a.prefix - 1, a.prefix - 1, a.c2, lds, D, D, src, st);
    }
  }
  // a page outside the cache: the waves load different rows, so all tell
  const bool any_bad = __syncthreads_or(bad != 0);
  const float l = any_bad ? __builtin_nanf("") : sum_across32(st.l);
  // own keys' weights are 2^score over a sum: of the prefix's weights as they are, since a rounding to bf16 that many
  // of them share is one of the sum (up to 2^-8 of it)
  float exact = 0.0f;
  if constexpr (kWeigh) exact = any_bad ? __builtin_nanf("") : sum_across32(st.exact);
  // the rows' partial sums by way of LDS (32 rows a wave, 16-byte chunk c of row n at c ^ n), so that a
  // store writes whole lines (16.8 MB of them: 0.8 us less than from the registers, 32 bytes
  // of a row at a time)
  constexpr int kChunks = D / 4;
  static_assert(kPreWaves * 32 * D * 4 <= flash_lds<D>(), "the rows fit the tiles' LDS");
  char* wl = lds + wave * 32 * D * 4;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<f32x4*>(wl + n * D * 4 + 16 * ((8 * dt + 2 * c + hf) ^ (n & (kChunks - 1)))) =
          f32x4{st.o[dt][4 * c], st.o[dt][4 * c + 1], st.o[dt][4 * c + 2], st.o[dt][4 * c + 3]};
  wave_fence();
  const int64_t at0 = (static_cast<int64_t>(split) * a.kv_heads + h) * rows + wr0;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const int row = i * (64 / kChunks) + lane / kChunks, c = lane % kChunks;
    if (wr0 + row < rows)
      *reinterpret_cast<f32x4*>(a.pre_o + (at0 + row) * D + 4 * c) =
          *reinterpret_cast<const f32x4*>(wl + row * D * 4 + 16 * (c ^ (row & (kChunks - 1))));
  }
  if (hf == 0 && wr0 + n < rows) {
    *reinterpret_cast<float2*>(a.pre_ml + (at0 + n) * 2) = float2{st.m, l};
    if constexpr (kWeigh) a.pre_l[at0 + n] = exact;
  }
}

template <int D, int RT, bool F8, bool kWeigh>
__global__ __launch_bounds__(kPgThreads, RT == 1 ? 2 : 1) void k_paged(const PagedArgs a) {
  __shared__ SegLds<D, RT, 4> lds;
  shares<D, RT, F8, kWeigh>(a, blockIdx.x, 16 * RT * blockIdx.y, lds);
}

// The prefix's workgroups, then the shares (more than 32 rows: a half of the rows each).
template <int D, int RT, bool F8, bool kWeigh>
__global__ __launch_bounds__(kPgThreads, RT == 1 ? 2 : 1) void k_paged_prefix(const PagedArgs a) {
  extern __shared__ __align__(16) char lds[];
  const int block = blockIdx.x - a.prefix_blocks;
  if (block < 0) prefix_part<D, F8, kWeigh>(a, blockIdx.x, lds);
  else shares<D, RT, F8, kWeigh>(a, block % a.shares, 16 * RT * (block / a.shares), *reinterpret_cast<SegLds<D, RT, 4>*>(lds));
}

// A workgroup for 16 rows of an item; nothing is left to join.  260 keys of 8 heads of 128 take 7.3
// us: the launch, length and page ids, keys, and the eight waves' parts through LDS, one
// after the other.
template <int D, bool F8, bool kWeigh>
__global__ __launch_bounds__(64 * kPgShortWaves, 2) void k_paged_short(const PagedArgs a) {
  __shared__ SegLds<D, 1, kPgShortWaves> lds;
  const int h = blockIdx.x % a.kv_heads, b = blockIdx.x / a.kv_heads, M = a.q_len * a.group, r0 = 16 * blockIdx.y;
  const int ids = page_ids<kPgShortWaves>(a, b, 0, 0);   // on its way beside the length
  bool bad_len;
  const int len = length_of(a, b, bad_len);
  if (len > 0) {
    segment<D, 1, kPgShortWaves, F8, kWeigh>(a, b, h, len, bad_len, r0, 0, len, -1, ids, lds);
    return;
  }
  for (int i = threadIdx.x; i < (min(M, r0 + 16) - r0) * (D / 8); i += 64 * kPgShortWaves) {
    const int r = r0 + i / (D / 8), tok = r / a.group, hd = h * a.group + r % a.group;
    *reinterpret_cast<u32x4*>(a.out + (static_cast<int64_t>(b) * a.q_len + tok) * a.o_token + hd * a.o_head + 8 * (i % (D / 8))) =
        u32x4{0u, 0u, 0u, 0u};
  }
}

// Joins a row's parts (shares of its own keys, splits of the prefix), WPR waves a
// row: their maxima and sums first, a part a lane, then groups of D / 4 lanes add up the
// parts in a fixed order.  Also writes the rows of sequences without keys.
// From kPgWaveRows rows on a wave each, since a workgroup then has little to do a row: 2048 rows of
// 18 parts of 128 take 6.6 us so, 7.4 with four waves (of 2 parts 5.3 either way); below, four
// waves: 256 rows of 17 parts of 64 take 4.9 us, with one 7.4.  Most of it is the launch and
// the loads after each other: length and place, maxima and sums beside the first parts.
constexpr int kPgWaveRows = 1024;

// Where the parts of the rows of item (b, h), whose sequence has len keys, lie among the partial rows.
struct Parts {
  int own, all, slot0;               // of its own keys; with the prefix's; the first of them
  int64_t pre, pre_step;             // rows of the prefix's first part, and from one to the next
  int M;
  bool done;                         // finished where it was computed: no parts
  __device__ __forceinline__ Parts(const PagedArgs& a, const i32x2& of_item, int b, int h, int len) {
    M = a.q_len * a.group;
    done = len > 0 && of_item.y == 0;
    // (kept inside the partial rows, also where a length has changed since the shares ran)
    slot0 = min(max(of_item.x, 0), 2 * a.shares + (a.splits ? a.batch * a.kv_heads : 0) - 1);
    own = len > 0 ? min(max(of_item.y, 1), max(a.shares - (slot0 >> 1), 1)) : 0;
    all = done ? 0 : own + a.splits;
    pre_step = static_cast<int64_t>(a.kv_heads) * a.batch * M;
    pre = static_cast<int64_t>(h) * a.batch * M + static_cast<int64_t>(b) * M;
  }
  // row r in part i: of a share its first (2 share) or last (2 share + 1) item, the
  // later parts are the first of theirs; parts >= own are the prefix's
  __device__ __forceinline__ int64_t row(int i, int r) const {
    if (i >= own) return (i - own) * pre_step + pre + r;
    return static_cast<int64_t>(i == 0 ? slot0 : (slot0 | 1) - 1 + 2 * i) * M + r;
  }
  // (the maximum alone: of a pair's load the register of the unused half is soon another value's, which then waits for the
  // load; the join of 8 x 2 tokens 5.2 us so, 4.6 now)
  __device__ __forceinline__ float top(const PagedArgs& a, int i, int r) const {
    return ldg<float>((i < own ? a.pml : a.pre_ml) + row(i, r) * 2);
  }
  __device__ __forceinline__ f32x2 ml(const PagedArgs& a, int i, int r) const {
    return ldg<f32x2>((i < own ? a.pml : a.pre_ml) + row(i, r) * 2);
  }
  // the sum of part i's weights before any rounding, its ml being `had`
  __device__ __forceinline__ float exact(const PagedArgs& a, int i, int r, const f32x2& had) const {
    return i < own ? had[1] : ldg<float>(a.pre_l + row(i, r));
  }
};

template <int D, int WPR, bool kWeigh>
__device__ __forceinline__ void join_rows(const PagedArgs& a, int block) {
  constexpr int kLanes = D / 4, kThreads = 64 * WPR, kWays = kThreads / kLanes, kRows = kPgThreads / kThreads;
  __shared__ float red[kRows][WPR], red_exact[kRows][WPR];
  __shared__ f32x4 sums[kRows][kWays][kLanes];
  const int M = a.q_len * a.group, tid = threadIdx.x % kThreads, lane = threadIdx.x & 63, wave = tid >> 6;
  const int mine = __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads), row = block * kRows + mine;
  const bool live = row < a.batch * a.kv_heads * M;
  const int r = row % M, item = row / M, h = item % a.kv_heads, b = live ? item / a.kv_heads : 0;
  const i32x2 of_item = ldg<i32x2>(a.parts + b * a.kv_heads + h);   // beside the length; nothing where there are no keys
  bool bad;
  const int len = length_of(a, b, bad);
  const Parts of(a, of_item, b, h, len);
  const bool done = of.done;
  if (WPR > 1 && done) return;
  const int own = of.own, parts = live ? of.all : 0;
  auto row_of = [&](int i) { return of.row(i, r); };
  auto ml_of = [&](int i) { return of.ml(a, i, r); };
  auto top_of = [&](int i) { return of.top(a, i, r); };
  // the first parts of every group of lanes, on their way beside the maxima and sums
  const int way = tid / kLanes, d0 = 4 * (tid % kLanes);
  auto part_of = [&](int i) { return ldg<f32x4>((i < own ? a.po : a.pre_o) + row_of(i) * D + d0); };
  constexpr int kAhead = 8 / WPR;
  f32x4 first[kAhead];
  float first_m[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const bool is = way + i * kWays < parts;
    first[i] = is ? part_of(way + i * kWays) : f32x4{0.f, 0.f, 0.f, 0.f};
    first_m[i] = is ? top_of(way + i * kWays) : kNegInf;
  }

  float top = kNegInf, ll = 0.0f, exact = 0.0f;
  for (int i = tid; i < parts; i += kThreads) top = fmaxf(top, top_of(i));
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
  if constexpr (WPR > 1) {
    if (lane == 0) red[mine][wave] = top;
    __syncthreads();
    top = red[mine][0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) top = fmaxf(top, red[mine][w]);
    __syncthreads();                                  // everyone has read the maxima
  }
  const float mu = top == kNegInf ? 0.0f : top;
  for (int i = tid; i < parts; i += kThreads) {
    const f32x2 ml = ml_of(i);
    ll += ml[1] * __builtin_amdgcn_exp2f(ml[0] - mu);
    if constexpr (kWeigh) exact += of.exact(a, i, r, ml) * __builtin_amdgcn_exp2f(ml[0] - mu);
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) {
    ll += __shfl_xor(ll, s, 64);
    if constexpr (kWeigh) exact += __shfl_xor(exact, s, 64);
  }
  if constexpr (WPR > 1) {
    if (lane == 0) {
      red[mine][wave] = ll;
      if constexpr (kWeigh) red_exact[mine][wave] = exact;
    }
    __syncthreads();
    ll = red[mine][0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) ll += red[mine][w];
    if constexpr (kWeigh) {
      exact = red_exact[mine][0];
#pragma unroll
      for (int w = 1; w < WPR; ++w) exact += red_exact[mine][w];
    }
  }
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (way + i * kWays < parts) y += first[i] * __builtin_amdgcn_exp2f(first_m[i] - mu);
#pragma unroll 4
  for (int i = way + kAhead * kWays; i < parts; i += kWays) y += part_of(i) * __builtin_amdgcn_exp2f(top_of(i) - mu);
  sums[mine][way][tid % kLanes] = y;
  if constexpr (WPR > 1) __syncthreads();
  else wave_fence();
  if (way || !live || done) return;
#pragma unroll
  for (int w = 1; w < kWays; ++w) y += sums[mine][w][tid % kLanes];
  const int tok = r / a.group, hd = h * a.group + r % a.group;
  // no key, or an unused slot (its q may hold anything): zeros
  const bool sees = a.lens[b] >= 0 && (a.prefix > 0 || len - a.q_len + tok >= 0 || ll != ll);
  if constexpr (kWeigh)
    if (d0 == 0) a.lse[static_cast<int64_t>(item) * M + r] = sees ? top + log2f(exact) : -kNegInf;
  y = sees ? y * (1.0f / ll) : f32x4{0.f, 0.f, 0.f, 0.f};
  *reinterpret_cast<u32x2*>(a.out + (static_cast<int64_t>(b) * a.q_len + tok) * a.o_token + hd * a.o_head + d0) =
      u32x2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
}

// Adds to every key's weight what the item's rows gave it, 2^(score - lse) of each, in a fixed order: kLanes lanes take
// a key's rows by fours, then a tree over them.  Workgroups of an item take its keys in turn.  M float32 a key and head
// are written by the scores' kernel and read here, against 4 D bytes of its key and value (2 D in 8 bits).
constexpr int kKwRows = 64;          // most rows of an item

// log2 of a row's sum of 2^score, by its parts: 16 lanes a row, for 16 rows.
constexpr int kKwPartRows = kPgThreads / 16;
__device__ __forceinline__ float lse_of_parts(const PagedArgs& a, const Parts& of, int b, int len) {
  const int r = threadIdx.x / 16, lane = threadIdx.x % 16;
  float top = kNegInf, l = 0.0f;     // l: of the weights before any rounding
  if (r < of.M)
    for (int i = lane; i < of.all; i += 16) top = fmaxf(top, of.top(a, i, r));
#pragma unroll
  for (int s = 8; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
  const float mu = top == kNegInf ? 0.0f : top;
  if (r < of.M)
    for (int i = lane; i < of.all; i += 16) {
      const f32x2 ml = of.ml(a, i, r);
      l += of.exact(a, i, r, ml) * __builtin_amdgcn_exp2f(ml[0] - mu);
    }
#pragma unroll
  for (int s = 8; s >= 1; s >>= 1) l += __shfl_xor(l, s, 64);
  const bool sees = a.lens[b] >= 0 && (a.prefix > 0 || len - a.q_len + r / a.group >= 0 || l != l);
  return sees ? top + log2f(l) : -kNegInf;
}

// kParts: rows in parts have no lse yet (the join is in the same launch), so it is made from the parts.
template <int kLanes, bool kParts>
__device__ __forceinline__ void weigh_keys(const PagedArgs& a, int block, int each) {
  constexpr int kKeys = kPgThreads / kLanes;
  __shared__ __align__(16) float lse[kKwRows];
  __shared__ __align__(16) int last[kKwRows];          // key that the row sees (-1: there is no such row)
  const int item = block / each, part = block % each, b = item / a.kv_heads, h = item % a.kv_heads, M = a.q_len * a.group;
  i32x2 of_item{};
  if constexpr (kParts) of_item = ldg<i32x2>(a.parts + item);
  bool bad;
  const int len = length_of(a, b, bad);
  if (bad || len <= part * kKeys) return;
  const Parts of(a, of_item, b, h, len);
  if (threadIdx.x < kKwRows)
    last[threadIdx.x] = static_cast<int>(threadIdx.x) < M ? len - a.q_len + static_cast<int>(threadIdx.x) / a.group : -1;
  if (kParts && !of.done) {
    const float x = lse_of_parts(a, of, b, len);
    if (threadIdx.x % 16 == 0) lse[threadIdx.x / 16] = x;
    if (static_cast<int>(threadIdx.x) >= kKwPartRows && threadIdx.x < kKwRows) lse[threadIdx.x] = -kNegInf;
  } else
  if (threadIdx.x < kKwRows)
    lse[threadIdx.x] = static_cast<int>(threadIdx.x) < M ? a.lse[static_cast<int64_t>(item) * M + threadIdx.x] : -kNegInf;
  __syncthreads();
  const int64_t cap = static_cast<int64_t>(a.c.max_pages) << a.c.page_shift;
  const int lane = threadIdx.x % kLanes, stride = (M + 3) & ~3;
  for (int key0 = part * kKeys; key0 < len; key0 += each * kKeys) {
    const int key = min(key0 + static_cast<int>(threadIdx.x) / kLanes, len - 1);   // (all lanes go on to the tree)
    const int id = ldg<int32_t>(a.c.table + b * a.c.table_stride + (key >> a.c.page_shift));
    const float* x = a.scores + (item * cap + key) * stride;
    float sum = 0.0f;
    for (int r = 4 * lane; r < M; r += 4 * kLanes) {
      const f32x4 v = ldg<f32x4>(x + r), e = *reinterpret_cast<const f32x4*>(&lse[r]);
      const i32x4 n = *reinterpret_cast<const i32x4*>(&last[r]);
#pragma unroll
      for (int i = 0; i < 4; ++i)                     // nothing of a key that the row does not see, whatever the row is
        if (key <= n[i]) sum += __builtin_amdgcn_exp2f(v[i] - e[i]);
    }
#pragma unroll
    for (int s = kLanes / 2; s >= 1; s >>= 1) sum += __shfl_xor(sum, s, 64);
    if (lane == 0 && key0 + static_cast<int>(threadIdx.x) / kLanes < len && id >= 0 && id < a.c.n_pages)
      a.weights[((static_cast<int64_t>(id) * a.kv_heads + h) << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1))] += sum;
  }
}

template <int D, int WPR, bool kWeigh>
__global__ __launch_bounds__(kPgThreads) void k_paged_join(const PagedArgs a) {
  join_rows<D, WPR, kWeigh>(a, blockIdx.x);
}
template <int kLanes>
__global__ __launch_bounds__(kPgThreads) void k_key_weights(const PagedArgs a, int each) {
  weigh_keys<kLanes, false>(a, blockIdx.x, each);
}
// Both in one launch, for up to kKwPartRows rows an item (48 sequences of up to 2100 keys, 4 rows: 21.7 us, 24.7 with two).
template <int D, int WPR, int kLanes>
__global__ __launch_bounds__(kPgThreads) void k_join_weights(const PagedArgs a, int each, int join_blocks) {
  const int block = blockIdx.x - join_blocks;
  if (block < 0) join_rows<D, WPR, false>(a, blockIdx.x);
  else weigh_keys<kLanes, true>(a, block, each);
}

// Workspace: partial rows of the shares (and, beside a prefix, of whole items), then the prefix's, then
// scores.
struct PagedPlan {
  int rt, shares, splits, row_tiles;
  bool alone;                        // k_paged_short
  size_t po, pml, parts, pre_o, pre_ml, scores, lse, pre_l, total;
};

PagedPlan plan_of(const dsk_paged_desc& d, const dsk_kv_cache& c, const PagedMore& more) {
  PagedPlan p{};
  auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
  const int64_t M = static_cast<int64_t>(d.q_len) * (d.heads / d.kv_heads);
  const int64_t items = static_cast<int64_t>(d.batch) * d.kv_heads, keys = static_cast<int64_t>(c.max_pages) * c.page_size;
  // With scales or weights, up to kPgFewKeys places of more than 16 rows: 16 rows a workgroup, two a CU, read the cache
  // once more but wait less.  8 key heads of 128, weights in 8 bits: one sequence of 8000 keys and three of 300, 64 rows, 35.1 us, 38.7 with 32 rows
  // a workgroup, 32 rows 32.5 and 35.4; four of 8000, 64 rows, 74.0 and 74.4; 64 of 4000, 32 rows, 335 and 315 (bf16: 602 and 412).
  const bool extra = more.f8 || more.weigh, few = extra && items * keys <= kPgFewKeys;
  p.rt = M <= 16 || few ? 1 : 2;
  // Up to kPgShort keys are two steps of a workgroup of eight waves, whose loads are all in flight at once: one
  // sequence with 8 key heads of 128 takes 7.3 us for 260 keys, with shares and their join
  // 9.3, but 9.9 against 9.3 for 517 and 14.6 against 9.3 for 1000.  Where items fill the
  // machine without shares, the join is all that they would add (64 such sequences of 600 / 1000 keys: 30.2 / 44.5 us, 31.6 / 45.9
  // with shares).
  // Codes take half the time, so up to 1024 places whatever the items.  Calls alone / with shares, us: 8 key heads of 128, one sequence of
  // 517 keys 10.1 / 12.2, 800 11.5 / 12.4, 1000 12.9 / 12.4; 16 of 1000 13.5 / 17.6; 48 of 800 23.3 / 23.1, of 1000 28.9 / 28.1; 4 key heads
  // of 64, one of 1000 9.7 / 12.3, 48 10.8 / 16.7.  With weights too, whose kernel waits for it, though few items then take longer (one
  // of 517 14.5 / 13.4, of 1000 17.5 / 13.4; 16 of 1000 19.4 / 21.2), since in 8 bits outputs are the same bits with and without weights.
  // (a launch counts its threads in 32 bits)
  p.alone = d.prefix_len == 0 && keys <= (items >= kPgMany || more.f8 ? kPgShortMany : kPgShort) &&
            items * (64 * kPgShortWaves) < (int64_t{1} << 32);
  p.total = 256;
  // behind what the call needs otherwise
  auto add_more = [&]() {
    if (more.weigh) {
      p.scores = p.total;
      p.lse = up(p.scores + static_cast<size_t>(items) * keys * ((M + 3) & ~int64_t{3}) * 4);
      p.pre_l = up(p.lse + static_cast<size_t>(items) * M * 4);
      p.total = up(p.pre_l + static_cast<size_t>(p.splits) * items * M * 4);
    }
    return p;
  };
  if (p.alone) return add_more();
  const int64_t units = items * ((keys + kPgUnit - 1) / kPgUnit + (more.f8 ? item_units<true>() : item_units<false>()));
  // the workgroups that are resident at once, two a CU (64 sequences of up to 8192 keys, 8 heads
  // of 128: 81 us, 90 with 256 and 86 with 768); one a CU where registers allow no
  // more, or beside a prefix's (36.5 us with 256, 39.4 with 512, 64 sequences behind 16385 keys)
  // (with scales or weights, workgroups for all rows of a share are resident at once: that sequence of 8000 keys with 64
  // rows takes 45.9 us with shares for one workgroup each, 35.1 with a quarter as many)
  const int64_t each = extra && (M > 32 || few) ? (M + 16 * p.rt - 1) / (16 * p.rt) : 1;
  const int64_t most = (p.rt == 1 && d.prefix_len == 0 ? 512 : 256) / each;
  p.shares = static_cast<int>(units < most ? units : most);
  const int64_t rows = static_cast<int64_t>(d.batch) * M;
  if (d.prefix_len > 0) {
    p.row_tiles = static_cast<int>((rows + kPreRows - 1) / kPreRows);
    const int64_t blocks = static_cast<int64_t>(p.row_tiles) * d.kv_heads, tiles = (d.prefix_len + kFlKeys - 1) / kFlKeys;
    const int64_t want = (kPreBlocks + blocks - 1) / blocks;
    // A split's time are its tiles, about 1 us each (heads of 128), and it adds partial rows to write and to
    // read, about 0.5 us for 2048 rows: least for the root of their ratio.  64 sequences
    // with 32 heads of 128 behind 4096 keys: 29.4 us with 8 splits, 34.5 with 16; behind 2000 keys 20.5
    // with 8, 23.5 with 16, 23.0 with 4; 16 sequences 17.8 with 32, 16.3 with 16, 17.0 with 8
    const double best = sqrt(4096.0 * static_cast<double>(tiles) / static_cast<double>(rows * d.kv_heads));
    const int64_t balanced = best < 1.0 ? 1 : static_cast<int64_t>(best + 0.5);
    p.splits = static_cast<int>(std::min({want, balanced, tiles}));
  }
  const size_t own = (2 * static_cast<size_t>(p.shares) + (p.splits ? items : 0)) * M;
  const size_t pre = static_cast<size_t>(p.splits) * d.kv_heads * rows;
  p.po = 0;
  p.pml = up(p.po + own * d.head_dim * 4);
  p.parts = up(p.pml + own * 8);
  p.pre_o = up(p.parts + items * 8);
  p.pre_ml = up(p.pre_o + pre * d.head_dim * 4);
  p.total = up(p.pre_ml + pre * 8);
  return add_more();
}

// Weights: lanes a key, workgroups an item, and whether they go with the join.  At least about kKwBlocks workgroups for a lane a key
// (of 16 lanes a key four times as many: 11.1 -> 9.3 us for 64 rows of four sequences of up to 8000 keys).
constexpr int kKwBlocks = 2048;
int weigh_lanes(int M) { return M <= 4 ? 1 : M <= 16 ? 4 : 16; }
int weigh_each(const PagedArgs& a, int M) {
  const int lanes = weigh_lanes(M), items = a.batch * a.kv_heads, keys = kPgThreads / lanes;
  const int of_row = ((a.c.max_pages << a.c.page_shift) + keys - 1) / keys;
  return std::min((kKwBlocks * (lanes == 16 ? 4 : lanes == 4 ? 2 : 1) + items - 1) / items, of_row);
}
bool weigh_beside_join(const PagedPlan& p, int M) { return !p.alone && M <= kKwPartRows; }

template <int D, int RT, bool F8, bool kWeigh>
void launch_paged_rt(const PagedPlan& p, const PagedArgs& a, hipStream_t s) {
  const int M = a.q_len * a.group;
  // more than 32 rows: every share (item) twice, a half of the rows each, which reads the cache twice (four row
  // tiles spill registers): 64 sequences of 4096 keys of one head of 128 take 40 us for 32 rows, 63 for 48, 65 for 64
  const int halves = (M + 16 * RT - 1) / (16 * RT);
  if (p.alone) {
    launch_kernel(k_paged_short<D, F8, kWeigh>, dim3(a.batch * a.kv_heads, (M + 15) / 16), 64 * kPgShortWaves, 0, s, a);
    return;
  }
  if (p.splits) {
    constexpr size_t lds = sizeof(SegLds<D, RT, 4>) > flash_lds<D>() ? sizeof(SegLds<D, RT, 4>) : flash_lds<D>();
    launch_kernel(k_paged_prefix<D, RT, F8, kWeigh>, a.prefix_blocks + p.shares * halves, kPgThreads, lds, s, a);
  } else {
    launch_kernel(k_paged<D, RT, F8, kWeigh>, dim3(p.shares, halves), kPgThreads, 0, s, a);
  }
  const int rows = a.batch * a.kv_heads * M;
  const bool waves = rows >= kPgWaveRows;
  const int blocks = waves ? (rows + 3) / 4 : rows;
  if constexpr (kWeigh)
    if (weigh_beside_join(p, M)) {
      const int lanes = weigh_lanes(M), each = weigh_each(a, M);
      auto kernel = lanes == 1 ? (waves ? k_join_weights<D, 1, 1> : k_join_weights<D, 4, 1>) : (waves ? k_join_weights<D, 1, 4> : k_join_weights<D, 4, 4>);
      launch_kernel(kernel, blocks + a.batch * a.kv_heads * each, kPgThreads, 0, s, a, each, blocks);
      return;
    }
  launch_kernel(waves ? k_paged_join<D, 1, kWeigh> : k_paged_join<D, 4, kWeigh>, blocks, kPgThreads, 0, s, a);
}

template <int D, bool F8, bool kWeigh>
void launch_paged_d(const PagedPlan& p, const PagedArgs& a, hipStream_t s) {
  if (p.rt == 1) launch_paged_rt<D, 1, F8, kWeigh>(p, a, s);
  else launch_paged_rt<D, 2, F8, kWeigh>(p, a, s);
  if constexpr (kWeigh) {
    const int M = a.q_len * a.group, lanes = weigh_lanes(M), each = weigh_each(a, M);
    if (!weigh_beside_join(p, M))
      launch_kernel(lanes == 1 ? k_key_weights<1> : lanes == 4 ? k_key_weights<4> : k_key_weights<16>, a.batch * a.kv_heads * each, kPgThreads,
                    0, s, a, each);
  }
}

}  // namespace

size_t paged_workspace(const dsk_paged_desc& d, const dsk_kv_cache& c, const PagedMore& more) { return plan_of(d, c, more).total; }

hipError_t launch_paged(const dsk_paged_desc& d, const dsk_kv_cache& c, const PagedMore& more, const void* q, const CacheView& view,
                        const int32_t* lens, const int32_t* prefix, void* out, void* ws, hipStream_t s) {
  const PagedPlan p = plan_of(d, c, more);
  char* w = static_cast<char*>(ws);
  const PagedArgs a{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(out), lens, view,
                    reinterpret_cast<float*>(w + p.po), reinterpret_cast<float*>(w + p.pml), reinterpret_cast<i32x2*>(w + p.parts),
                    reinterpret_cast<float*>(w + p.pre_o), reinterpret_cast<float*>(w + p.pre_ml), prefix,
                    d.q_token, d.q_head, d.o_token, d.o_head, d.scale * kLog2e, d.batch, d.q_len, d.kv_heads,
                    d.heads / d.kv_heads, d.prefix_len, p.shares, p.splits, p.row_tiles,
                    p.row_tiles * p.splits * d.kv_heads, more.k_scale, more.v_scale, more.key_weights, reinterpret_cast<float*>(w + p.scores),
                    reinterpret_cast<float*>(w + p.lse), reinterpret_cast<float*>(w + p.pre_l)};
  auto form = [&](auto f8, auto weigh) {
    constexpr bool kF = decltype(f8)::value, kW = decltype(weigh)::value;
    if (d.head_dim == 64) launch_paged_d<64, kF, kW>(p, a, s);
    else launch_paged_d<128, kF, kW>(p, a, s);
  };
  if (more.f8) more.weigh ? form(std::true_type{}, std::true_type{}) : form(std::true_type{}, std::false_type{});
  else more.weigh ? form(std::false_type{}, std::true_type{}) : form(std::false_type{}, std::false_type{});
  return hipGetLastError();
}

}  // namespace dsk
