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
#include <math.h>

#include <algorithm>

#include "attn_core.h"

namespace dsk {
namespace {

constexpr int kPgThreads = 256;
constexpr int kPgUnit = 128;        // keys of a unit: 32 for each of four waves
constexpr int kPgShort = 512;       // keys of a table row that one workgroup takes alone
constexpr int kPgShortMany = 1024;  // where there are kPgMany items
constexpr int kPgMany = 512;
constexpr int kPgShortWaves = 8;

typedef int i32x2 __attribute__((ext_vector_type(2)));
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
};

// Keys of sequence b that the cache can hold; `bad` if lens[b] claims more.
__device__ __forceinline__ int length_of(const PagedArgs& a, int b, bool& bad) {
  const int n = a.lens[b], cap = a.c.max_pages << a.c.page_shift;
  bad = n > cap;
  return min(max(n, 0), cap);
}
__device__ __forceinline__ int units_of(const PagedArgs& a, int b) {
  bool bad;
  return (length_of(a, b, bad) + kPgUnit - 1) / kPgUnit;
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
__device__ __forceinline__ Units units_at(const PagedArgs& a, int b0) {
  const int b = b0 + (threadIdx.x & 63);
  const uint32_t n = b < a.batch ? units_of(a, b) : 0;
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

template <int D>
struct Step {                       // one wave's 32 keys
  u32x4 k[2][D / 32];
  uint32_t v[8][D / 32];            // VW = D / 16 elements of 8 keys
};

template <int VW>
__device__ __forceinline__ void load_v(uint32_t (&v)[VW / 2], const uint16_t* p) {
  if constexpr (VW == 8) {
    const u32x4 r = ldg16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r[i];
  } else {
    const u32x2 r = ldg<u32x2>(p);
    v[0] = r[0];
    v[1] = r[1];
  }
}

// LDS of a segment of W waves: their rows, then maxima and sums.
template <int D, int RT, int W>
struct SegLds {
  float o[W][16][D + 4];
  float ml[W][16 * RT][2];
};

// Lane 2 i + kt: the page of the wave's 16-key tile kt in step kk + i (the table row's
// last one behind its end; the sequence's length need not be known yet).
template <int W>
__device__ __forceinline__ int page_ids(const PagedArgs& a, int b, int kk) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tile = (static_cast<int64_t>(kk) + (lane >> 1)) * (2 * W) + 2 * wave + (lane & 1);
  const int page = static_cast<int>(min(tile >> (a.c.page_shift - 4), static_cast<int64_t>(a.c.max_pages - 1)));
  return ldg<int32_t>(a.c.table + b * a.c.table_stride + page);
}

// Units [k0, k1) of the keys of item (b, h), in units of 32 W keys, for the rows from
// r0 on: to `out` (slot < 0: they are all of the item's) or to the partial rows of `slot`.
// first_ids: page_ids of k0.
template <int D, int RT, int W>
__device__ __forceinline__ void segment(const PagedArgs& a, int b, int h, int len, bool bad_len, int r0, int k0, int k1,
                                        int64_t slot, int first_ids, SegLds<D, RT, W>& lds) {
  constexpr int VW = D / 16, KS = D / 32, kUnit = 32 * W;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  const int M = a.q_len * a.group;
    // queries: column n16 of row tile rt is row 16 rt + n16 = token * group + head of the group
    bf16x8 q[RT][KS];
    int lim[RT];                    // last key that the lane's row sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = min(r0 + 16 * rt + n16, M - 1), tok = r / a.group, hd = h * a.group + r % a.group;
      const uint16_t* p = a.q + (static_cast<int64_t>(b) * a.q_len + tok) * a.q_token + hd * a.q_head + 8 * g;
      lim[rt] = len - a.q_len + tok;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) q[rt][ks] = as_bf16x8(ldg16(p + 32 * ks));
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
    const int last_tile = (len - 1) >> 4;
    int ids = first_ids, ids0 = k0;   // lane 2 i + kt: the page of tile kt of step ids0 + i
    int bad_tile = INT32_MAX;         // the lane's first 16 keys on a page outside the cache
    auto check_ids = [&]() {
      const int step = ids0 + (lane >> 1), tile = step * (2 * W) + 2 * wave + (lane & 1);
      const bool out_of = ids < 0 || ids >= a.c.n_pages;
      if (out_of && step < k1 && tile <= last_tile) bad_tile = min(bad_tile, tile);
      if (out_of) ids = 0;
    };
    check_ids();
    auto load = [&](Step<D>& s, int kk) {
      if (kk - ids0 >= 32) {
        ids0 = kk;
        ids = page_ids<W>(a, b, kk);
        check_ids();
      }
      const int tile0 = kk * (2 * W) + 2 * wave;
      if (tile0 > last_tile) return;                  // none of the wave's keys in this step
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int tile = min(tile0 + kt, last_tile);
        const int id = __builtin_amdgcn_readlane(ids, 2 * (kk - ids0) + tile - tile0);
        const int last_row = len - 1 - tile * 16;     // rows past the length: the last one again
        const int row0 = (tile * 16) & ((1 << a.c.page_shift) - 1);
        const int64_t base = (((static_cast<int64_t>(id) * a.kv_heads + h) << a.c.page_shift) + row0) * D;
        const uint16_t* kp = a.c.k + base + min(n16, last_row) * D + 8 * g;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s.k[kt][ks] = ldg16(kp + 32 * ks);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          load_v<VW>(s.v[4 * kt + j], a.c.v + base + min(4 * g + j, last_row) * D + VW * n16);
      }
    };
    // rarely: infinite and NaN values of step kk, to the rows that see them (the
    // products then leave them out)
    auto add_nonfinite = [&](int kk) {
#pragma unroll 1
      for (int key = kk * kUnit + 32 * wave, end = min(key + 32, len); key < end; ++key) {
        int id = ldg<int32_t>(trow + (key >> a.c.page_shift));
        if (id < 0 || id >= a.c.n_pages) id = 0;
        const int in_page = key & ((1 << a.c.page_shift) - 1);
        const uint16_t* vp = a.c.v + (((static_cast<int64_t>(id) * a.kv_heads + h) << a.c.page_shift) + in_page) * D;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int t = 0; t < VW; ++t) {
            const float x = nonfinite_only(ldg<uint16_t>(vp + VW * (4 * g + r) + t));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][t][r] += key <= lim[rt] ? x : 0.0f;
          }
      }
    };
    auto compute = [&](const Step<D>& s, int kk) {
      const int key0 = kk * kUnit + 32 * wave;
      if (key0 >= len) return;
      const bool masked = key0 + 31 > len - a.q_len;
      bf16x8 p[RT], rest[RT];         // the weights: bf16, and what that rounds off
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 x[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          x[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) x[kt] = mfma16(as_bf16x8(s.k[kt][ks]), q[rt][ks], x[kt]);
        }
        if (masked) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (key0 + 16 * kt + 4 * g + r > lim[rt]) x[kt][r] = kNegInf;
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
      // An infinite value times a weight's rest, which may be zero or negative, or the weight zero of a key that a
      // row does not see or of a place behind the last key (that key's values again), would be NaN: are
      // all the values finite?  The largest exponents of the pairs tell (decode_64 0.5 us more than without).
      u16x2 largest = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < VW / 2; ++i)
          largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16x2, s.v[j][i] & 0x7f807f80u));
      const bool finite = !__any(nonfinite_bits(__builtin_bit_cast(uint32_t, largest)) != 0);
      if (!finite) add_nonfinite(kk);
#pragma unroll
      for (int t = 0; t < VW; ++t) {
        const uint32_t sel = t & 1 ? 0x07060302u : 0x05040100u;
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(s.v[2 * i + 1][t / 2], s.v[2 * i][t / 2], sel);
        if (!finite)
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = finite_only(w[i]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][t] = mfma16(as_bf16x8(w), rest[rt], mfma16(as_bf16x8(w), p[rt], o[rt][t]));
      }
    };

    Step<D> s0, s1;
    load(s0, k0);
    int kk = k0;
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
template <int D, int RT>
__device__ __forceinline__ void shares(const PagedArgs& a, int share, int r0, SegLds<D, RT, 4>& lds) {
  Units n;
  uint32_t all = 0;                  // units of one key head
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    n = units_at(a, b0);
    all += lane_value(n.up_to, 63);
  }
  const uint32_t total = all * a.kv_heads, quota = (total + a.shares - 1) / a.shares;
  const uint32_t u0 = share * quota, u1 = min(u0 + quota, total);
  if (u0 >= u1) return;
  // the sequence that u0 lies in, and the units of one key head in those before it
  const uint32_t first_unit = u0 / a.kv_heads;
  uint32_t before = 0;
  int b = a.batch;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) n = units_at(a, b0);
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
    const uint32_t nb = (len + kPgUnit - 1) / kPgUnit, first = before * a.kv_heads;
    if (nb == 0 || u >= first + nb * a.kv_heads) {
      before += nb;
      ++b;
      continue;
    }
    // an item's first unit is kv_heads * before + h * its units
    const int h = static_cast<int>((u - first) / nb);
    const uint32_t item0 = first + h * nb;
    const int k0 = static_cast<int>(u - item0), k1 = static_cast<int>(min(nb, u1 - item0));
    const bool whole = k0 == 0 && k1 == static_cast<int>(nb);
    const int64_t slot = whole ? (a.splits ? 2 * static_cast<int64_t>(a.shares) + static_cast<int64_t>(b) * a.kv_heads + h : -1)
                               : 2 * static_cast<int64_t>(share) + (u == u0 ? 0 : 1);
    if (k0 == 0 && r0 == 0 && threadIdx.x == 0)
      a.parts[b * a.kv_heads + h] =
          i32x2{static_cast<int>(slot), whole ? (a.splits ? 1 : 0) : static_cast<int>((item0 + nb - 1) / quota) - share + 1};
    segment<D, RT, 4>(a, b, h, len, bad_len, r0, k0, k1, slot, page_ids<4>(a, b, k0), lds);
    u = item0 + k1;
  }
}

// All rows of the batch against a part of the prefix: tile `row_tile` of 128 rows of
// head h, split `split` of the keys.
constexpr int kPreWaves = 4;
constexpr int kPreRows = 32 * kPreWaves;
constexpr int kPreBlocks = 256;      // workgroups of the prefix, at most about: one a CU (prefix of 16385 keys for 64
                                     // sequences: 40 us, 45 with 128, 47 with 384, 50 with 512)
constexpr int kPreChunk = 64;        // tiles whose places in the cache a wave holds at once

template <int D>
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
  st.l = 0.0f;
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
    auto src = [&](int t, int row, const uint16_t*& kp, const uint16_t*& vp, int& last) {
      const uint32_t lo = __builtin_amdgcn_readlane(at_lo, t - c0), hi = __builtin_amdgcn_readlane(at_hi, t - c0);
      const int64_t base = static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
      kp = a.c.k + base;
      vp = a.c.v + base;
      last = max(a.prefix - 1 - (t * kFlKeys + row), 0);
    };
    if (c0 > t0) __syncthreads();      // the last chunk's reads of LDS are done
    flash<D, kPreWaves, 1>(q, c0, c1, a.prefix - 1, a.prefix - 1, a.prefix - 1, a.c2, lds, D, D, src, st);
  }
  // a page outside the cache: the waves load different rows, so all tell
  const bool any_bad = __syncthreads_or(bad != 0);
  const float l = any_bad ? __builtin_nanf("") : sum_across32(st.l);
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
  if (hf == 0 && wr0 + n < rows) *reinterpret_cast<float2*>(a.pre_ml + (at0 + n) * 2) = float2{st.m, l};
}

template <int D, int RT>
__global__ __launch_bounds__(kPgThreads, RT == 1 ? 2 : 1) void k_paged(const PagedArgs a) {
  __shared__ SegLds<D, RT, 4> lds;
  shares<D, RT>(a, blockIdx.x, 16 * RT * blockIdx.y, lds);
}

// The prefix's workgroups, then the shares (more than 32 rows: a half of the rows each).
template <int D, int RT>
__global__ __launch_bounds__(kPgThreads, RT == 1 ? 2 : 1) void k_paged_prefix(const PagedArgs a) {
  extern __shared__ __align__(16) char lds[];
  const int block = blockIdx.x - a.prefix_blocks;
  if (block < 0) prefix_part<D>(a, blockIdx.x, lds);
  else shares<D, RT>(a, block % a.shares, 16 * RT * (block / a.shares), *reinterpret_cast<SegLds<D, RT, 4>*>(lds));
}

// A workgroup for 16 rows of an item; nothing is left to join.  260 keys of 8 heads of 128 take 7.3
// us: the launch, length and page ids, keys, and the eight waves' parts through LDS, one
// after the other.
template <int D>
__global__ __launch_bounds__(64 * kPgShortWaves, 2) void k_paged_short(const PagedArgs a) {
  __shared__ SegLds<D, 1, kPgShortWaves> lds;
  constexpr int kUnit = 32 * kPgShortWaves;
  const int h = blockIdx.x % a.kv_heads, b = blockIdx.x / a.kv_heads, M = a.q_len * a.group, r0 = 16 * blockIdx.y;
  const int ids = page_ids<kPgShortWaves>(a, b, 0);   // on its way beside the length
  bool bad_len;
  const int len = length_of(a, b, bad_len);
  if (len > 0) {
    segment<D, 1, kPgShortWaves>(a, b, h, len, bad_len, r0, 0, (len + kUnit - 1) / kUnit, -1, ids, lds);
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

template <int D, int WPR>
__global__ __launch_bounds__(kPgThreads) void k_paged_join(const PagedArgs a) {
  constexpr int kLanes = D / 4, kThreads = 64 * WPR, kWays = kThreads / kLanes, kRows = kPgThreads / kThreads;
  __shared__ float red[kRows][WPR];
  __shared__ f32x4 sums[kRows][kWays][kLanes];
  const int M = a.q_len * a.group, tid = threadIdx.x % kThreads, lane = threadIdx.x & 63, wave = tid >> 6;
  const int mine = __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads), row = blockIdx.x * kRows + mine;
  const bool live = row < a.batch * a.kv_heads * M;
  const int r = row % M, item = row / M, h = item % a.kv_heads, b = live ? item / a.kv_heads : 0;
  const i32x2 of_item = ldg<i32x2>(a.parts + b * a.kv_heads + h);   // beside the length; nothing where there are no keys
  bool bad;
  const int len = length_of(a, b, bad);
  const bool done = len > 0 && of_item.y == 0;        // finished where it was computed
  if (WPR > 1 && done) return;
  // (kept inside the partial rows, also where a length has changed since the shares ran)
  const int slot0 = min(max(of_item.x, 0), 2 * a.shares + (a.splits ? a.batch * a.kv_heads : 0) - 1);
  const int own = len > 0 ? min(max(of_item.y, 1), max(a.shares - (slot0 >> 1), 1)) : 0;
  const int parts = !live || done ? 0 : own + a.splits;
  // row of part i among the partial rows: of a share its first (2 share) or last (2 share + 1) item, the
  // later parts are the first of theirs; parts >= own are the prefix's
  auto row_of = [&](int i) -> int64_t {
    if (i >= own)
      return (static_cast<int64_t>(i - own) * a.kv_heads + h) * (static_cast<int64_t>(a.batch) * M) + static_cast<int64_t>(b) * M + r;
    return static_cast<int64_t>(i == 0 ? slot0 : (slot0 | 1) - 1 + 2 * i) * M + r;
  };
  auto ml_of = [&](int i) { return ldg<f32x2>((i < own ? a.pml : a.pre_ml) + row_of(i) * 2); };
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
    first_m[i] = is ? ml_of(way + i * kWays)[0] : kNegInf;
  }

  float top = kNegInf, ll = 0.0f;
  for (int i = tid; i < parts; i += kThreads) top = fmaxf(top, ml_of(i)[0]);
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
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) ll += __shfl_xor(ll, s, 64);
  if constexpr (WPR > 1) {
    if (lane == 0) red[mine][wave] = ll;
    __syncthreads();
    ll = red[mine][0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) ll += red[mine][w];
  }
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (way + i * kWays < parts) y += first[i] * __builtin_amdgcn_exp2f(first_m[i] - mu);
#pragma unroll 4
  for (int i = way + kAhead * kWays; i < parts; i += kWays) y += part_of(i) * __builtin_amdgcn_exp2f(ml_of(i)[0] - mu);
  sums[mine][way][tid % kLanes] = y;
  if constexpr (WPR > 1) __syncthreads();
  else wave_fence();
  if (way || !live || done) return;
#pragma unroll
  for (int w = 1; w < kWays; ++w) y += sums[mine][w][tid % kLanes];
  const int tok = r / a.group, hd = h * a.group + r % a.group;
  // no key, or an unused slot (its q may hold anything): zeros
  const bool sees = a.lens[b] >= 0 && (a.prefix > 0 || len - a.q_len + tok >= 0 || ll != ll);
  y = sees ? y * (1.0f / ll) : f32x4{0.f, 0.f, 0.f, 0.f};
  *reinterpret_cast<u32x2*>(a.out + (static_cast<int64_t>(b) * a.q_len + tok) * a.o_token + hd * a.o_head + d0) =
      u32x2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
}

// Workspace: partial rows of the shares (and, beside a prefix, of whole items), then the prefix's.
struct PagedPlan {
  int rt, shares, splits, row_tiles;
  bool alone;                        // k_paged_short
  size_t po, pml, parts, pre_o, pre_ml, total;
};

PagedPlan plan_of(const dsk_paged_desc& d, const dsk_kv_cache& c) {
  PagedPlan p{};
  auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
  const int64_t M = static_cast<int64_t>(d.q_len) * (d.heads / d.kv_heads);
  p.rt = M <= 16 ? 1 : 2;
  const int64_t items = static_cast<int64_t>(d.batch) * d.kv_heads, keys = static_cast<int64_t>(c.max_pages) * c.page_size;
  // Up to kPgShort keys are two steps of a workgroup of eight waves, whose loads are all in flight at once: one
  // sequence with 8 key heads of 128 takes 7.3 us for 260 keys, with shares and their join
  // 9.3, but 9.9 against 9.3 for 517 and 14.6 against 9.3 for 1000.  Where items fill the
  // machine without shares, the join is all that they would add (64 such sequences of 600 / 1000 keys: 30.2 / 44.5 us, 31.6 / 45.9
  // with shares).
  // (a launch counts its threads in 32 bits)
  p.alone = d.prefix_len == 0 && keys <= (items >= kPgMany ? kPgShortMany : kPgShort) &&
            items * (64 * kPgShortWaves) < (int64_t{1} << 32);
  p.total = 256;
  if (p.alone) return p;
  const int64_t units = items * ((keys + kPgUnit - 1) / kPgUnit);
  // the workgroups that are resident at once, two a CU (64 sequences of up to 8192 keys, 8 heads
  // of 128: 81 us, 90 with 256 and 86 with 768); one a CU where registers allow no
  // more, or beside a prefix's (36.5 us with 256, 39.4 with 512, 64 sequences behind 16385 keys)
  const int64_t most = p.rt == 1 && d.prefix_len == 0 ? 512 : 256;
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
  return p;
}

template <int D, int RT>
void launch_paged_rt(const PagedPlan& p, const PagedArgs& a, hipStream_t s) {
  const int M = a.q_len * a.group;
  // more than 32 rows: every share (item) twice, a half of the rows each, which reads the cache twice (four row
  // tiles spill registers): 64 sequences of 4096 keys of one head of 128 take 40 us for 32 rows, 63 for 48, 65 for 64
  const int halves = (M + 16 * RT - 1) / (16 * RT);
  if (p.alone) {
    launch_kernel(k_paged_short<D>, dim3(a.batch * a.kv_heads, (M + 15) / 16), 64 * kPgShortWaves, 0, s, a);
    return;
  }
  if (p.splits) {
    constexpr size_t lds = sizeof(SegLds<D, RT, 4>) > flash_lds<D>() ? sizeof(SegLds<D, RT, 4>) : flash_lds<D>();
    launch_kernel(k_paged_prefix<D, RT>, a.prefix_blocks + p.shares * halves, kPgThreads, lds, s, a);
  } else {
    launch_kernel(k_paged<D, RT>, dim3(p.shares, halves), kPgThreads, 0, s, a);
  }
  const int rows = a.batch * a.kv_heads * M;
  if (rows >= kPgWaveRows) launch_kernel(k_paged_join<D, 1>, (rows + 3) / 4, kPgThreads, 0, s, a);
  else launch_kernel(k_paged_join<D, 4>, rows, kPgThreads, 0, s, a);
}

}  // namespace

size_t paged_workspace(const dsk_paged_desc& d, const dsk_kv_cache& c) { return plan_of(d, c).total; }

hipError_t launch_paged(const dsk_paged_desc& d, const dsk_kv_cache& c, const void* q, const CacheView& view,
                        const int32_t* lens, const int32_t* prefix, void* out, void* ws, hipStream_t s) {
  const PagedPlan p = plan_of(d, c);
  char* w = static_cast<char*>(ws);
  const PagedArgs a{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(out), lens, view,
                    reinterpret_cast<float*>(w + p.po), reinterpret_cast<float*>(w + p.pml), reinterpret_cast<i32x2*>(w + p.parts),
                    reinterpret_cast<float*>(w + p.pre_o), reinterpret_cast<float*>(w + p.pre_ml), prefix,
                    d.q_token, d.q_head, d.o_token, d.o_head, d.scale * kLog2e, d.batch, d.q_len, d.kv_heads,
                    d.heads / d.kv_heads, d.prefix_len, p.shares, p.splits, p.row_tiles,
                    p.row_tiles * p.splits * d.kv_heads};
  if (d.head_dim == 64) {
    if (p.rt == 1) launch_paged_rt<64, 1>(p, a, s);
    else launch_paged_rt<64, 2>(p, a, s);
  } else {
    if (p.rt == 1) launch_paged_rt<128, 1>(p, a, s);
    else launch_paged_rt<128, 2>(p, a, s);
  }
  return hipGetLastError();
}

}  // namespace dsk
