// Norms of queries and keys for each head, their rotation, and the append to a
// paged cache, in one pass.
//
// One head row is D elements, held by D / 8 lanes with 8 consecutive elements
// each, so a row is read and written in 16-byte pieces (bf16) and its mean of
// squares is a tree over 8 or 16 lanes.  The rotation of element e needs its
// pair's other element: interleaved pairs lie in the lane's own 8; of half
// pairs the lane reads the other 8 elements too (a second load of a line that
// is on its way already, instead of eight lane exchanges).
//
// Angles: position * freq[i] turns by millions of radians at far positions,
// where float32 has no digit of the fraction left.  The product is formed in
// float64, its whole turns are taken off there, and the remaining fraction of a
// turn (error below 2^-50 position) goes to float32.
//
// One wave a token, its heads in turn, so that what belongs to the token is made
// once: each lane computes a pair's sine and cosine (exchanged through LDS) and
// keeps its 8 elements' factors, gamma cos and +-gamma' sin, in registers.  A
// head then takes two multiply-adds an element, and the traffic bounds the
// kernel: 8192 tokens of 32 + 8 + 8 heads of 128 into a cache take 36 us (5.6
// TB/s), 4095 of 32 + 8 20 us (4.2 TB/s); a block for four tokens with the factors
// from LDS for every head took 53 and 28 us.  Few tokens: a token's heads over
// several waves, queries apart from keys and values, for the latency.
#include <type_traits>

#include "attn.h"

namespace dsk {
namespace {

constexpr int kQkWaves = 4;            // of a workgroup, a token each
constexpr int kQkAhead = 4;            // heads of a group of lanes whose loads are in flight together
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));   // gammas may start anywhere

struct QkArgs {
  const void *q, *k, *v;
  const int32_t *positions, *seq;
  const double* freq;
  const float *q_gamma, *k_gamma;
  uint16_t *q_out, *k_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, qo_token, qo_head, ko_token, ko_head;
  int32_t tokens, heads, kv_heads, rot_dim, rot_first, prefix_len, norm;
  int32_t q_parts, kv_parts;         // waves of a token for queries, and for keys and values (kAll: one for all)
  float eps, mscale;
  CacheView cache;
  bool append;
};

// 8 elements as they lie in memory.
template <bool kBF16>
struct Raw8 {
  u32x4 v[kBF16 ? 1 : 2];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (kBF16) {
      v[0] = ldg16(static_cast<const uint16_t*>(p) + i);
    } else {
      const float* f = static_cast<const float*>(p) + i;
      v[0] = ldg16(f);
      v[1] = ldg16(f + 4);
    }
  }
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (kBF16) return __uint_as_float(j & 1 ? v[0][j >> 1] & 0xffff0000u : v[0][j >> 1] << 16);
    else return __uint_as_float(v[j >> 2][j & 3]);
  }
};

// A lane's part of a head row: elements e .. e + 7 of 8 lanes (D 64) or 16 (D 128).  kAll: a
// wave takes all heads of its token.  kPast: queries and rows of the cache are written past L2.
template <int D, bool kBF16, bool kInter, bool kAll, bool kPast>
__global__ __launch_bounds__(64 * kQkWaves) void k_qk(const QkArgs a) {
  constexpr int kLanes = D / 8, kRows = 64 / kLanes;  // lanes of a head row, rows of a wave
  __shared__ float2 turns[kQkWaves][D / 2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wl = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kQkWaves + wave;
  if (t >= a.tokens) return;
  const int lane = wl % kLanes, e = 8 * lane;
  const int half = a.rot_dim / 2, er = e - a.rot_first;       // this lane's first element among the rotated
  const bool rotated = er >= 0 && er < a.rot_dim, low = er < half;
  // half pairs: the elements that pair with the lane's own
  const int ep = kInter || !rotated ? e : (low ? e + half : e - half);
  // this lane's heads: row0, row0 + step, ..
  const bool is_q = kAll || static_cast<int>(blockIdx.y) < a.q_parts;
  const int part = is_q ? blockIdx.y : blockIdx.y - a.q_parts;
  const int row0 = part * kRows + wl / kLanes, step = (kAll ? 1 : is_q ? a.q_parts : a.kv_parts) * kRows;

  // heads row, row + step, .. of one tensor: kQkAhead of them
  struct Heads { Raw8<kBF16> x[kQkAhead], y[kQkAhead]; };
  auto load = [&](Heads& r, const void* p, int64_t token, int64_t head, int row, int rows, bool pairs) {
#pragma unroll
    for (int i = 0; i < kQkAhead; ++i) {
      const int64_t at = t * token + min(row + i * step, rows - 1) * head;
      r.x[i].load(p, at + e);
      if (!kInter && pairs) r.y[i].load(p, at + ep);
    }
  };
  // the first heads, in flight beside the angles
  Heads r, v;
  if (is_q && row0 < a.heads) load(r, a.q, a.q_token, a.q_head, row0, a.heads, true);
  if (!is_q && row0 < a.kv_heads) {
    load(r, a.k, a.k_token, a.k_head, row0, a.kv_heads, true);
    if (a.append) load(v, a.v, a.v_token, a.v_head, row0, a.kv_heads, false);
  }

  const int pos = a.positions[t];
  if (pos < 0) return;                                // a token of padding
  float2* turn = turns[wave];
  if (wl < half) {
    double c = static_cast<double>(pos) * (a.freq[wl] * 0.15915494309189533577);   // turns: / (2 pi)
    c -= rint(c);
    float sn, cs;
    sincospif(2.0f * static_cast<float>(c), &sn, &cs);
    turn[wl] = float2{cs * a.mscale, sn * a.mscale};
  }
  // the token's row of the cache, or none
  int64_t slot = -1;
  if (a.append) {
    const int sq = a.seq[t];
    const int64_t at = static_cast<int64_t>(pos) - a.prefix_len, page = at >> a.cache.page_shift;
    if (sq >= 0 && sq < a.cache.n_seqs && at >= 0 && page < a.cache.max_pages) {
      const int id = a.cache.table[sq * a.cache.table_stride + page];
      if (id >= 0 && id < a.cache.n_pages)
        slot = ((static_cast<int64_t>(id) * a.kv_heads) << a.cache.page_shift) + (at & ((1 << a.cache.page_shift) - 1));
    }
  }

  // own[j] x[j] + pair[j] y[j] is element j, before the norm's factor: gamma alone where
  // nothing turns, gamma cos and -+gamma' sin (interleaved: of the lane's other element) where it does
  auto factors = [&](const float* gamma, float (&own)[8], float (&pair)[8]) {
    float g[8], gp[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = gp[j] = 1.0f;
    if (gamma) {
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const f32x4 u = *reinterpret_cast<const f32x4_a4*>(gamma + e + j), v = *reinterpret_cast<const f32x4_a4*>(gamma + ep + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) { g[j + i] = u[i]; gp[j + i] = v[i]; }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int pr = kInter ? er / 2 + j / 2 : (low ? er : er - half) + j;
      const float2 cs = rotated ? turn[pr] : float2{1.0f, 0.0f};
      own[j] = g[j] * cs.x;
      if constexpr (kInter) pair[j] = j & 1 ? g[j - 1] * cs.y : -(g[j + 1] * cs.y);
      else pair[j] = (low ? -cs.y : cs.y) * gp[j];
    }
  };
  auto normed = [&](const Raw8<kBF16>& x, const Raw8<kBF16>& y, const float (&own)[8], const float (&pair)[8]) {
    float rstd = 1.0f, z[8];
    if (a.norm) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
      for (int m = kLanes / 2; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
      rstd = rsqrtf(ss * (1.0f / D) + a.eps);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // the other one's product only where something turns: it may be infinite
      const float other = kInter ? x[j ^ 1] : y[j];
      z[j] = x[j] * own[j];
      if (rotated) z[j] += other * pair[j];
      z[j] *= rstd;
    }
    return u32x4{pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3]), pack_bf16(z[4], z[5]), pack_bf16(z[6], z[7])};
  };

  auto store = [&](uint16_t* p, const u32x4& x) {
    if constexpr (kPast) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p));
    else *reinterpret_cast<u32x4*>(p) = x;
  };
  // each wave reads its own angles alone: its LDS writes are done before
  __builtin_amdgcn_wave_barrier();
  float own[8], pair[8];
  if (is_q && a.heads > 0) {
    factors(a.q_gamma, own, pair);
    for (int row = row0; row < a.heads;) {
      u32x4 out[kQkAhead];
#pragma unroll
      for (int i = 0; i < kQkAhead; ++i) out[i] = normed(r.x[i], r.y[i], own, pair);
      const int next = row + kQkAhead * step;
      // the next heads' loads before these stores; q_out may be q, since a head is read
      // whole before it is written
      if (next < a.heads) load(r, a.q, a.q_token, a.q_head, next, a.heads, true);
#pragma unroll
      for (int i = 0; i < kQkAhead; ++i)
        if (row + i * step < a.heads)
          store(a.q_out + t * a.qo_token + (row + i * step) * a.qo_head + e, out[i]);
      row = next;
    }
  }
  if (row0 >= a.kv_heads || (is_q && !kAll)) return;
  if (kAll) {
    load(r, a.k, a.k_token, a.k_head, row0, a.kv_heads, true);
    if (slot >= 0) load(v, a.v, a.v_token, a.v_head, row0, a.kv_heads, false);
  }
  factors(a.k_gamma, own, pair);
  for (int row = row0; row < a.kv_heads;) {
    u32x4 out[kQkAhead];
#pragma unroll
    for (int i = 0; i < kQkAhead; ++i) out[i] = normed(r.x[i], r.y[i], own, pair);
    const int next = row + kQkAhead * step;
    if (next < a.kv_heads) load(r, a.k, a.k_token, a.k_head, next, a.kv_heads, true);
#pragma unroll
    for (int i = 0; i < kQkAhead; ++i) {
      const int h = row + i * step;
      if (h >= a.kv_heads) break;
      if (a.k_out) *reinterpret_cast<u32x4*>(a.k_out + t * a.ko_token + h * a.ko_head + e) = out[i];   // read many times next
      if (slot >= 0) {
        const int64_t to = (slot + (static_cast<int64_t>(h) << a.cache.page_shift)) * D + e;
        store(a.cache.k + to, out[i]);
        const Raw8<kBF16>& x = v.x[i];
        store(a.cache.v + to, u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])});
      }
    }
    if (next < a.kv_heads && slot >= 0) load(v, a.v, a.v_token, a.v_head, next, a.kv_heads, false);
    row = next;
  }
}

// Calls that write this many bytes write queries and rows of the cache past L2: on tensors of its own each,
// 32 + 8 + 8 heads of 128, 512 tokens (6 MB) take 7.0 -> 6.6 us, 1024 10.6 -> 7.9, 2048 18.4 -> 16.4, 8192 49.2 -> 46.8, and with the prompt
// attention behind them 19.8 -> 19.0, 30.6 -> 29.3, 63.1 -> 63.3, 563 -> 566; 12 + 12 + 12 of 64, 1500 tokens (6.6 MB) 8.0 -> 7.2, 26.3 ->
// 25.5; 64 + 8 + 8 of 128, 2048 tokens 25.2 -> 23.4, 105 -> 110.  Fewer are read next and stay: 512 tokens of 16 + 4 + 4 heads
// of 64 (1.5 MB) 5.0 either way, 14.7 -> 14.9; 256 of 12 + 12 + 12 (1.1 MB) 12.8 -> 13.0.  k_out's rows, which the attention
// reads for every row tile, always stay: past L2 they cost it up to 16 % (3000 tokens of 12 + 12 + 12: 43.9 -> 50.5).
constexpr int64_t kPastL2 = 4 << 20;

template <int D>
void launch_qk_d(const dsk_qk_desc& d, const QkArgs& args, hipStream_t s) {
  constexpr int kRows = 64 / (D / 8);
  // Few tokens: a token's heads over several waves, kQkAhead heads to a group of lanes (1024 tokens, whole ones
  // against those: 32 + 8 + 8 heads of 128 11.0 and 7.9 us, 12 + 12 + 12 of 64 7.5 and 5.9, 4 + 1 + 1 8.2 and 5.4; 2048: 15.7 and
  // 14.7, 8.5 and 9.4, 8.3 and 9.9; 8192: 45.7 and 50.8, 28.0 and 29.1, 19.8 and 22.2).  Without queries there is little to
  // spread (16 tokens 4.4 and 4.5, 2048 6.6 and 6.7).
  const int per = kRows * kQkAhead;
  const bool split = d.tokens < 2048 && d.heads > 0;
  const int q_parts = split ? (d.heads + per - 1) / per : 0, kv_parts = split ? (d.kv_heads + per - 1) / per : 0;
  QkArgs a = args;
  a.q_parts = q_parts;
  a.kv_parts = kv_parts;
  const dim3 grid((d.tokens + kQkWaves - 1) / kQkWaves, split ? q_parts + kv_parts : 1);
  const int64_t rows = static_cast<int64_t>(d.tokens) * (d.heads + (a.k_out ? d.kv_heads : 0) + (a.append ? 2 * d.kv_heads : 0));
  const bool past = rows * D * 2 >= kPastL2;
  auto launch = [&](auto whole, auto parts, auto whole_past, auto parts_past) {
    launch_kernel(past ? (split ? parts_past : whole_past) : (split ? parts : whole), grid, 64 * kQkWaves, 0, s, a);
  };
  auto form = [&](auto bf16, auto inter) {
    constexpr bool kB = decltype(bf16)::value, kI = decltype(inter)::value;
    launch(k_qk<D, kB, kI, true, false>, k_qk<D, kB, kI, false, false>, k_qk<D, kB, kI, true, true>, k_qk<D, kB, kI, false, true>);
  };
  if (d.dtype == DSK_DTYPE_BF16) {
    if (d.interleaved) form(std::true_type{}, std::true_type{});
    else form(std::true_type{}, std::false_type{});
  } else {
    if (d.interleaved) form(std::false_type{}, std::true_type{});
    else form(std::false_type{}, std::false_type{});
  }
}

}  // namespace

hipError_t launch_qk(const dsk_qk_desc& d, const void* q, const void* k, const void* v, const int32_t* positions,
                     const int32_t* seq, const double* freq, const float* q_gamma, const float* k_gamma,
                     const CacheView* cache, void* q_out, void* k_out, hipStream_t s) {
  QkArgs a{q, k, v, positions, seq, freq, q_gamma, k_gamma, static_cast<uint16_t*>(q_out),
           static_cast<uint16_t*>(k_out), d.q_token, d.q_head, d.k_token, d.k_head, d.v_token, d.v_head,
           d.qo_token, d.qo_head, d.ko_token, d.ko_head, d.tokens, d.heads, d.kv_heads, d.rot_dim, d.rot_first,
           d.prefix_len, d.norm, 0, 0, d.eps, d.mscale, cache ? *cache : CacheView{}, cache != nullptr};
  if (d.head_dim == 64) launch_qk_d<64>(d, a, s);
  else launch_qk_d<128>(d, a, s);
  return hipGetLastError();
}

}  // namespace dsk
