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
//
// Keys and values for a cache in 8 bits: a block's scale needs the largest element of all its rows, so
// a workgroup takes the tokens of whole blocks (append_codes), beside those of the
// queries in one launch: 8192 tokens of 32 + 8 + 8 heads of 128 take 43 us (4.3 TB/s), 64 of them 6.6.
#include <type_traits>

#include "kv8.h"

namespace dsk {
namespace {

constexpr int kQkWaves = 4;            // of a workgroup, a token each
constexpr int kQkAhead = 4;            // heads of a group of lanes whose loads are in flight together
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));   // gammas may start anywhere

struct QkArgs {
  const void *q, *k, *v;
  const int32_t *positions, *seq;
  const int32_t *axis, *rows;        // axis of each pair, cache row of each token, or null
  int64_t axis_stride;
  const double* freq;
  const float *q_gamma, *k_gamma;
  uint16_t *q_out, *k_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, qo_token, qo_head, ko_token, ko_head;
  int32_t tokens, heads, kv_heads, rot_dim, rot_first, prefix_len, norm;
  int32_t q_parts, kv_parts;         // waves of a token for queries, and for keys and values (kAll: one for all)
  float eps, mscale;
  CacheView cache;
  bool append;
  int32_t n_axes;
  float* key_weights;                // of the cache's rows, or null
  uint8_t *k_scale, *v_scale;        // of a cache in 8 bits
  int32_t windows, code_parts;       // workgroups for it: of kWindow tokens, times parts of the heads
};

// kMore: the call may have several axes, rows of its own or weights.

// Whether token t, at pos on the first axis, is one of padding.
template <bool kMore>
__device__ __forceinline__ bool left_out(const QkArgs& a, int64_t t, int pos) {
  bool out = pos < 0;
  if constexpr (kMore)
    for (int x = 1; x < a.n_axes; ++x) out |= a.positions[x * a.axis_stride + t] < 0;
  return out;
}
// Cosine and sine of pair i's angle, times mscale; a pair of no axis does not turn.  kFine: quarter turns are taken off in
// float64 too, so that the rest is at most an eighth and loses up to two bits less.  For codes, which are
// off by a whole step where the key's own error crosses a border (16 times 8192 tokens: 187 such codes, 342 without, 43.4 us
// either way).
template <bool kFine, bool kMore>
__device__ __forceinline__ float2 turn_of(const QkArgs& a, int64_t t, int pos, int i) {
  if (kMore && a.axis) {
    const int x = a.axis[i];
    pos = x >= 0 && x < a.n_axes ? a.positions[x * a.axis_stride + t] : 0;
  }
  double c = static_cast<double>(pos) * (a.freq[i] * 0.15915494309189533577);   // turns: / (2 pi)
  c -= rint(c);
  float sn, cs;
  if constexpr (kFine) {
    const double n = rint(4.0 * c);
    const int quarter = static_cast<int>(n);
    float x, y;
    sincospif(2.0f * static_cast<float>(c - 0.25 * n), &y, &x);
    cs = quarter & 1 ? -y : x;
    sn = quarter & 1 ? x : y;
    if (quarter & 2) { cs = -cs; sn = -sn; }
  } else {
    sincospif(2.0f * static_cast<float>(c), &sn, &cs);
  }
  return float2{cs * a.mscale, sn * a.mscale};
}
// Row of token t among all rows of the cache with one head, or -1.
template <bool kMore>
__device__ __forceinline__ int64_t slot_of(const QkArgs& a, int64_t t, int pos) {
  const int sq = a.seq[t];
  const int64_t at = kMore && a.rows ? a.rows[t] : static_cast<int64_t>(pos) - a.prefix_len, page = at >> a.cache.page_shift;
  if (sq < 0 || sq >= a.cache.n_seqs || at < 0 || page >= a.cache.max_pages) return -1;
  const int id = a.cache.table[sq * a.cache.table_stride + page];
  if (id < 0 || id >= a.cache.n_pages) return -1;
  return ((static_cast<int64_t>(id) * a.kv_heads) << a.cache.page_shift) + (at & ((1 << a.cache.page_shift) - 1));
}

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

// The rotation as a lane sees it: its elements e .. e + 7, and those that pair with them.
template <bool kInter>
struct Pairs {
  int e, er, ep, half;
  bool rotated, low;
  __device__ __forceinline__ Pairs(const QkArgs& a, int lane) {
    e = 8 * lane;
    half = a.rot_dim / 2;
    er = e - a.rot_first;                             // this lane's first element among the rotated
    rotated = er >= 0 && er < a.rot_dim;
    low = er < half;
    ep = kInter || !rotated ? e : (low ? e + half : e - half);   // half pairs: the elements that pair with the lane's own
  }
  // own[j] x[j] + pair[j] y[j] is element j, before the norm's factor: gamma alone where
  // nothing turns, gamma cos and -+gamma' sin (interleaved: of the lane's other element) where it does
  __device__ __forceinline__ void factors(const float* gamma, const float2* turn, float (&own)[8], float (&pair)[8]) const {
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
      // (read whether it turns or not, since a branch around each read waits for it: 8192 tokens 44.2 -> 43.1 us)
      const int pr = kInter ? er / 2 + j / 2 : (low ? er : er - half) + j;
      const float2 read = turn[rotated ? pr : 0], cs = rotated ? read : float2{1.0f, 0.0f};
      own[j] = g[j] * cs.x;
      if constexpr (kInter) pair[j] = j & 1 ? g[j - 1] * cs.y : -(g[j + 1] * cs.y);
      else pair[j] = (low ? -cs.y : cs.y) * gp[j];
    }
  }
};
// Eight elements of a head row that D / 8 lanes hold, normed and rotated.
template <int D, bool kBF16, bool kInter>
__device__ __forceinline__ void norm_turn(bool norm, float eps, bool rotated, const Raw8<kBF16>& x, const Raw8<kBF16>& y, const float (&own)[8],
                                          const float (&pair)[8], float (&z)[8]) {
  float rstd = 1.0f;
  if (norm) {
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
    for (int m = D / 16; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
    rstd = rsqrtf(ss * (1.0f / D) + eps);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // the other one's product only where something turns: it may be infinite
    const float other = kInter ? x[j ^ 1] : y[j];
    z[j] = x[j] * own[j];
    if (rotated) z[j] += other * pair[j];
    z[j] *= rstd;
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&z)[8]) {
  return u32x4{pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3]), pack_bf16(z[4], z[5]), pack_bf16(z[6], z[7])};
}

// Keys and values of a cache in 8 bits.  The tokens of a call that go to one block of 16 rows stand
// next to each other; the workgroup of the first one's window of 16 tokens takes them all (kSlots: up to
// 15 behind its window).  (With another token between them, also one that is left out, two take the block at once, and its
// scale and codes may be of either.)  A row lies in D / 8 lanes as elsewhere, its largest magnitude goes to the
// block's by way of LDS, and with that the block's scale is known before a code is made.
constexpr int kWindow = 16, kSlots = 2 * kWindow;

template <int D>
struct CodeLds {
  float2 turn[kSlots][D / 2];
  int64_t slot[kSlots];
  int lead[kSlots];                  // first token of the block; kSkip, or kCopy: for k_out alone
  uint32_t rows[kSlots];             // of the block that begins here: its rows that the call brings
  uint32_t top[3][2][kSlots];        // largest magnitudes, of three heads in turn
  int begin, end;                    // the slots from the first to the last that have something to do
};
constexpr int kSkip = -1, kCopy = -2;

template <int D, bool kBF16, bool kInter>
__device__ __forceinline__ void append_codes(const QkArgs& a, int block) {
  __shared__ CodeLds<D> s;
  constexpr int kLanes = D / 8, kRows = 64 * kQkWaves / kLanes, kPasses = kSlots / kRows;
  const int tid = threadIdx.x, lane = tid % kLanes, part = block % a.code_parts;
  const int64_t t0 = static_cast<int64_t>(block / a.code_parts) * kWindow;
  if (tid < 64) {                    // lane 1 + i: token t0 + i
    const int i = tid - 1;
    const int64_t t = t0 + i;
    int64_t slot = -1;
    bool live = false;
    if (i < kSlots && t >= 0 && t < a.tokens) {
      const int pos = a.positions[t];
      live = !left_out<true>(a, t, pos);
      if (live) slot = slot_of<true>(a, t, pos);
    }
    const int64_t key = slot < 0 ? -1 : slot / kScaleRows, before = __shfl_up(key, 1, 64);
    const uint64_t starts = __ballot(tid > 0 && (key < 0 || key != before));
    const uint64_t mine = starts & ((2ull << tid) - 1);
    const int first = mine ? 62 - __clzll(static_cast<long long>(mine)) : -1;
    const int lead = i < 0 || i >= kSlots ? kSkip : key >= 0 ? (first >= 0 && first < kWindow ? first : kSkip) : live && i < kWindow ? kCopy : kSkip;
    const uint64_t busy = __ballot(lead != kSkip);    // bit 1 + i
    if (i >= 0 && i < kSlots) {
      s.slot[i] = slot;
      s.rows[i] = 0;
      s.lead[i] = lead;
    }
    if (tid == 0) {
      s.begin = busy ? __ffsll(static_cast<long long>(busy)) - 2 : 0;
      s.end = busy ? 63 - __clzll(static_cast<long long>(busy)) : 0;
    }
  } else {
    for (int i = tid - 64; i < 3 * 2 * kSlots; i += 64 * (kQkWaves - 1)) (&s.top[0][0][0])[i] = 0;
  }
  __syncthreads();
  if (tid < kSlots && s.lead[tid] >= 0) atomicOr(&s.rows[s.lead[tid]], 1u << (s.slot[tid] & (kScaleRows - 1)));
  // (a prompt's blocks begin anywhere in its windows, and are 16 slots from there: one pass of rows)
  const int half = a.rot_dim / 2, begin = s.begin, end = s.end;
  if (begin >= end) return;
  for (int i = tid; i < (end - begin) * half; i += 64 * kQkWaves) {
    const int slot = begin + i / half;
    if (s.lead[slot] != kSkip) s.turn[slot][i % half] = turn_of<true, true>(a, t0 + slot, a.positions[t0 + slot], i % half);
  }
  __syncthreads();
  const Pairs<kInter> pairs(a, lane);
  const int passes = end - begin > kRows ? kPasses : 1;
  struct Row {
    int lead, own;                   // slots of the block's first row and of this one
    int64_t row;                     // of the cache, of the head in work
    const char *k, *v;               // the head's rows
    uint16_t* k_out;
    float own_f[8], pair_f[8];
  } rows[kPasses];
  const int size = kBF16 ? 2 : 4;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int i = begin + p * kRows + tid / kLanes;
    Row& r = rows[p];
    r.own = i;
    r.lead = i < end ? s.lead[i] : kSkip;
    if (r.lead == kSkip) continue;
    const int64_t t = t0 + i;
    r.row = s.slot[i] + (static_cast<int64_t>(part) << a.cache.page_shift);
    r.k = static_cast<const char*>(a.k) + (t * a.k_token + part * a.k_head) * size;
    r.v = static_cast<const char*>(a.v) + (t * a.v_token + part * a.v_head) * size;
    r.k_out = a.k_out ? a.k_out + t * a.ko_token + part * a.ko_head : nullptr;
    pairs.factors(a.k_gamma, s.turn[i], r.own_f, r.pair_f);
  }
  // a head's rows, on their way beside the work on the head before
  struct Loaded { Raw8<kBF16> x, y, v; int byte[2]; } raw[kPasses];
  auto load = [&](int p, const Row& r) {
    raw[p].x.load(r.k, pairs.e);
    if (!kInter) raw[p].y.load(r.k, pairs.ep);
    if (r.lead >= 0) {
      raw[p].v.load(r.v, pairs.e);
      raw[p].byte[0] = a.k_scale[r.row / kScaleRows];
      raw[p].byte[1] = a.v_scale[r.row / kScaleRows];
    }
  };
#pragma unroll
  for (int p = 0; p < kPasses; ++p)
    if (p < passes && rows[p].lead != kSkip) load(p, rows[p]);
  int buffer = 0;
  for (int h = part; h < a.kv_heads; h += a.code_parts, buffer = buffer == 2 ? 0 : buffer + 1) {
    float z[kPasses][2][8];          // keys, values
    int old[kPasses][2];
    bool odd[kPasses];               // of this lane's elements one is not finite
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      Row& r = rows[p];
      if (p >= passes || r.lead == kSkip) continue;   // (all lanes of a row alike)
      norm_turn<D, kBF16, kInter>(a.norm, a.eps, pairs.rotated, raw[p].x, raw[p].y, r.own_f, r.pair_f, z[p][0]);
      if (r.k_out) *reinterpret_cast<u32x4*>(r.k_out + pairs.e) = pack8(z[p][0]);
      if (r.lead >= 0) {
        odd[p] = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[p][1][j] = raw[p].v[j];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          // magnitudes as whole numbers: their order, with what is not finite above
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(z[p][w][j]) & 0x7fffffffu);
          if (top >= 0x7f800000u) {                   // rarely: without those
            odd[p] = true;
            top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t u = __float_as_uint(z[p][w][j]) & 0x7fffffffu;
              if (u < 0x7f800000u) top = max(top, u);
            }
          }
#pragma unroll
          for (int m = kLanes / 2; m >= 1; m >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, 64)));
          if (lane == 0) atomicMax(&s.top[buffer][w][r.lead], top);
          old[p][w] = min(raw[p].byte[w], 254);
        }
      }
      if (h + a.code_parts < a.kv_heads) {            // the next head
        r.k += a.code_parts * a.k_head * size;
        r.v += a.code_parts * a.v_head * size;
        if (r.k_out) r.k_out += a.code_parts * a.ko_head;
        r.row += static_cast<int64_t>(a.code_parts) << a.cache.page_shift;
        load(p, r);
      }
    }
    __syncthreads();
    // those of the head after next: read before the barrier above, used behind the next
    if (tid < 2 * kSlots) (&s.top[buffer == 0 ? 2 : buffer - 1][0][0])[tid] = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const Row& r = rows[p];
      if (p >= passes || r.lead < 0) continue;
      const int64_t row = s.slot[r.own] + (static_cast<int64_t>(h) << a.cache.page_shift);
      const uint32_t here = s.rows[r.lead];
      const bool fresh = here & 1;
      if (a.key_weights && lane == 0) a.key_weights[row] = 0.0f;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint8_t* codes = reinterpret_cast<uint8_t*>(w ? a.cache.v : a.cache.k);
        const int want = scale_byte(__uint_as_float(s.top[buffer][w][r.lead])), b = fresh ? want : max(want, old[p][w]);
        *reinterpret_cast<u32x2*>(codes + row * D + pairs.e) = to_codes(z[p][w], inverse_scale(b), odd[p] || b >= kMostScale);
        if (r.own != r.lead) continue;
        if (lane == 0) (w ? a.v_scale : a.k_scale)[row / kScaleRows] = static_cast<uint8_t>(b);
        if (fresh || b <= old[p][w]) continue;
        // the block's other rows, in the larger scale
        const float f = scale_step(old[p][w], b);
        uint8_t* block = codes + row / kScaleRows * kScaleRows * D + pairs.e;
        for (int i = 0; i < kScaleRows; ++i) {
          if (here >> i & 1) continue;
          u32x2* c = reinterpret_cast<u32x2*>(block + i * D);
          *c = u32x2{rescale4((*c)[0], f), rescale4((*c)[1], f)};
        }
      }
    }
  }
}

// A lane's part of a head row: elements e .. e + 7 of 8 lanes (D 64) or 16 (D 128).  kAll: a
// wave takes all heads of its token.  kPast: queries and rows of the cache are written past L2.
// kCodes: a cache in 8 bits, whose workgroups come first; then the queries'.  Plain calls have a form without kMore, which
// asks nothing about what they do not have (8192 tokens 43.3 -> 43.1 us).
template <int D, bool kBF16, bool kInter, bool kAll, bool kPast, bool kCodes, bool kMore>
__global__ __launch_bounds__(64 * kQkWaves) void k_qk(const QkArgs a) {
  constexpr int kLanes = D / 8, kRows = 64 / kLanes;  // lanes of a head row, rows of a wave
  __shared__ float2 turns[kQkWaves][D / 2];
  int bx = blockIdx.x, by = blockIdx.y;
  if constexpr (kCodes) {
    bx -= a.windows * a.code_parts;
    if (bx < 0) {
      append_codes<D, kBF16, kInter>(a, blockIdx.x);
      return;
    }
    by = bx % a.q_parts;
    bx /= a.q_parts;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wl = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(bx) * kQkWaves + wave;
  if (t >= a.tokens) return;
  const int lane = wl % kLanes;
  const Pairs<kInter> pairs(a, lane);
  const int e = pairs.e, ep = pairs.ep, er = pairs.er, half = pairs.half;
  const bool rotated = pairs.rotated, low = pairs.low;
  // this lane's heads: row0, row0 + step, ..
  const bool is_q = kAll || kCodes || by < a.q_parts;
  const int part = is_q ? by : by - a.q_parts;
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
  if (left_out<kMore>(a, t, pos)) return;
  float2* turn = turns[wave];
  if (wl < half) turn[wl] = turn_of<false, kMore>(a, t, pos, wl);
  const int64_t slot = !kCodes && a.append ? slot_of<kMore>(a, t, pos) : -1;   // the token's row of the cache, or none

  // as pairs.factors, written out with a branch around the reads of the angles, which is faster for a cache in bf16 (8192 tokens 42.4
  // us, 43.2 with pairs.factors, 44.1 with that and the branch; in 8 bits 43.8, 43.3 with pairs.factors)
  auto factors = [&](const float* gamma, float (&own)[8], float (&pair)[8]) {
    if constexpr (kCodes) {
      pairs.factors(gamma, turn, own, pair);
      return;
    }
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
    float z[8];
    norm_turn<D, kBF16, kInter>(a.norm, a.eps, rotated, x, y, own, pair, z);
    return pack8(z);
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
  if (kCodes || row0 >= a.kv_heads || (is_q && !kAll)) return;
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
        if (kMore && a.key_weights && lane == 0) a.key_weights[to / D] = 0.0f;
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

// Workgroups for the keys and values of a cache in 8 bits, at least about: heads of a token apart until there are these, though
// each makes the angles anew (8192 tokens 43.4 us, 46.9 with 1024, 54 with 2048).
constexpr int kCodeBlocks = 512;

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
    if (!a.k_scale) {
      auto rows = [&](auto more) {
        constexpr bool kM = decltype(more)::value;
        launch(k_qk<D, kB, kI, true, false, false, kM>, k_qk<D, kB, kI, false, false, false, kM>, k_qk<D, kB, kI, true, true, false, kM>,
               k_qk<D, kB, kI, false, true, false, kM>);
      };
      if (a.axis || a.rows || a.key_weights) rows(std::true_type{});
      else rows(std::false_type{});
      return;
    }
    a.windows = (d.tokens + kWindow - 1) / kWindow;
    const int want = (kCodeBlocks + a.windows - 1) / a.windows;
    a.code_parts = want < d.kv_heads ? want : d.kv_heads;
    if (!split) a.q_parts = d.heads > 0 ? 1 : 0;
    const int64_t blocks = static_cast<int64_t>(a.windows) * a.code_parts + static_cast<int64_t>(grid.x) * a.q_parts;
    launch_kernel(past ? k_qk<D, kB, kI, false, true, true, true> : k_qk<D, kB, kI, false, false, true, true>, dim3(static_cast<uint32_t>(blocks)),
                  64 * kQkWaves, 0, s, a);
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
                     const CacheView* cache, const QkMore& more, void* q_out, void* k_out, hipStream_t s) {
  QkArgs a{q, k, v, positions, seq, more.axis, more.rows, more.axis_stride, freq, q_gamma, k_gamma, static_cast<uint16_t*>(q_out),
           static_cast<uint16_t*>(k_out), d.q_token, d.q_head, d.k_token, d.k_head, d.v_token, d.v_head,
           d.qo_token, d.qo_head, d.ko_token, d.ko_head, d.tokens, d.heads, d.kv_heads, d.rot_dim, d.rot_first,
           d.prefix_len, d.norm, 0, 0, d.eps, d.mscale, cache ? *cache : CacheView{}, cache != nullptr,
           more.n_axes, more.key_weights, more.k_scale, more.v_scale, 0, 0};
  if (d.head_dim == 64) launch_qk_d<64>(d, a, s);
  else launch_qk_d<128>(d, a, s);
  return hipGetLastError();
}

}  // namespace dsk
