// Attention over packed prompts.
//
// The rows of a tile are (token, head of the group) pairs of one key head,
// token by token: the heads of a group share every key tile that is loaded, a
// short prompt of a few tokens fills a tile with its heads, and the causal edge
// crosses few keys of a tile.
//
// 8192 tokens of 32 + 8 heads of 128 take 474 to 515 us (1.16 to 1.07 PFLOP/s, by the
// card), bound by the products and the vector work beside them (flash).  16 ragged prompts
// of 5375 tokens together, 16 + 4 heads of 64, take 25.7 us of which the machine's
// work is 13: the longest prompt's last rows are 24 tiles in a row, and a CU that
// holds two such workgroups takes 24 us for them.  17 tokens take 6 us: the launch, the
// sequence bounds, then q and the first keys, one after the other.
#include "attn_core.h"

namespace dsk {
namespace {

constexpr int kFlWaves = 4;
constexpr int kFlThreads = 64 * kFlWaves;
constexpr int kFlRows = 32 * kFlWaves;
constexpr int kCus = 256;
constexpr int64_t kFewElements = 1 << 22;   // of K and of V: 8 MB each
constexpr int kMostRank = 1 << 23;   // of a sequence's first tile; tiles are at most 2^23

struct PromptArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  const int32_t *cu_q, *cu_k;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  float c2;
  int32_t tokens, kv_tokens, n_seqs, kv_heads, group, causal;
  int32_t first;                    // tiles whose workgroups (one a key head) come to a CU each
};

// A sequence's rows, cut to the tensors (whatever cu holds, no row outside is
// touched), and a row tile's place in it.
struct TilePlace { int q0, q1, k0, k1, at; };

// Row tile `tile` of all (false: there are fewer), the most keys first, 64 sequences at a
// time: tile i of a sequence has rank lo + i, lo for the keys before its first query, and
// those of a high rank come first.  The rank is searched for by 64 lanes at once.
// Workgroups are dealt out to the CUs in turn (the 257th comes to the first one's), so the
// second of a CU is taken in the opposite order: 8192 tokens of 16 heads of 64 / 128 take 163 /
// 262 us, 170 / 273 without, 4096 of 128 80 against 85.
template <int ROWS>
__device__ __forceinline__ bool find_tile(const PromptArgs& a, int tile, TilePlace& p) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < a.n_seqs; b0 += 64) {
    const int b = min(b0 + lane, a.n_seqs - 1), here = min(a.n_seqs - b0, 64);
    const int q0 = min(max(a.cu_q[b], 0), a.tokens), q1 = min(max(a.cu_q[b + 1], q0), a.tokens);
    const int k0 = min(max(a.cu_k[b], 0), a.kv_tokens), k1 = min(max(a.cu_k[b + 1], k0), a.kv_tokens);
    const int n = lane < here ? ((q1 - q0) * a.group + ROWS - 1) / ROWS : 0;
    const int before = a.causal ? max(k1 - k0 - (q1 - q0), 0) : k1 - k0;
    const int lo = min(before / ROWS, kMostRank / a.group) * a.group, hi = lo + n;
    auto from = [&](int rank) {                      // tiles of at least that rank
      int c = 0;
      for (int j = 0; j < here; ++j)
        c += min(max(__builtin_amdgcn_readlane(hi, j) - rank, 0), __builtin_amdgcn_readlane(n, j));
      return c;
    };
    int step = !__any(hi > 64) ? 1 : !__any(hi > 4096) ? 64 : !__any(hi > 262144) ? 4096 : 262144;
    int count = from(lane * step), rank = 0, above = 0;   // above: tiles of a higher rank
    const int all = __builtin_amdgcn_readfirstlane(count);
    if (tile >= all) {
      tile -= all;
      continue;
    }
    if (a.n_seqs <= 64 && tile >= a.first && tile < 2 * a.first) tile = a.first + min(2 * a.first, all) - 1 - tile;
    for (;;) {
      const int l = 63 - __clzll(__ballot(count > tile));  // lane 0 always
      rank += l * step;
      if (l < 63) above = __builtin_amdgcn_readlane(count, l + 1);
      if (step == 1) break;
      step /= 64;
      count = from(rank + lane * step);
    }
    // the sequences that have such a tile, in their order
    uint64_t have = __ballot(rank >= lo && rank < hi);
    for (int i = tile - above; i > 0; --i) have &= have - 1;
    const int l = __ffsll(static_cast<unsigned long long>(have)) - 1;
    p.q0 = __builtin_amdgcn_readlane(q0, l);
    p.q1 = __builtin_amdgcn_readlane(q1, l);
    p.k0 = __builtin_amdgcn_readlane(k0, l);
    p.k1 = __builtin_amdgcn_readlane(k1, l);
    p.at = rank - __builtin_amdgcn_readlane(lo, l);
    return true;
  }
  return false;
}

// KH waves for every 32 rows.
template <int D, int KH>
__global__ __launch_bounds__(kFlThreads, 2) void k_prompt(const PromptArgs a) {
  extern __shared__ __align__(16) char lds[];
  constexpr int ROWS = kFlRows / KH, RW = kFlWaves / KH;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hf = lane >> 5;
  const int h = blockIdx.x % a.kv_heads;
  TilePlace sr;
  if (!find_tile<ROWS>(a, static_cast<int>(blockIdx.x / a.kv_heads), sr)) return;
  const int lq = sr.q1 - sr.q0, lk = sr.k1 - sr.k0, rows = lq * a.group;
  const int row0 = sr.at * ROWS, wr0 = row0 + 32 * (wave % RW);
  const int r = min(wr0 + n, rows - 1), tok = r / a.group, hd = h * a.group + r % a.group;
  const int shift = lk - lq;                        // query i sees the keys up to i + shift
  const int lim = a.causal ? tok + shift : lk - 1;
  const int w_min = a.causal ? min(wr0, rows - 1) / a.group + shift : lk - 1;
  const int b_min = a.causal ? row0 / a.group + shift : lk - 1;
  const int b_last = min(row0 + ROWS - 1, rows - 1) / a.group;
  const int t1 = ((a.causal ? b_last + shift : lk - 1) + kFlKeys) / kFlKeys;   // <= 0 where no key is seen

  bf16x8 q[D / 16];
  const uint16_t* qp = a.q + (sr.q0 + static_cast<int64_t>(tok)) * a.q_token + hd * a.q_head + 8 * hf;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) q[ks] = as_bf16x8(ldg16(qp + 16 * ks));
  FlashRows<D> st;
  st.m = kNegInf;
  st.l = 0.0f;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) st.o[dt] = f32x16{};

  const uint16_t* kb = a.k + sr.k0 * a.k_token + h * a.k_head;
  const uint16_t* vb = a.v + sr.k0 * a.v_token + h * a.v_head;
  auto src = [&](int t, int row, const uint16_t*& kp, const uint16_t*& vp, int& last) {
    // rows past the sequence's end (another one's, or none): its last row again
    const int key = min(t * kFlKeys + row, lk - 1);
    kp = kb + key * a.k_token;
    vp = vb + key * a.v_token;
    last = lk - 1 - key;
  };
  flash<D, kFlWaves, KH>(q, 0, t1, lim, w_min, b_min, a.c2, lds, a.k_token, a.v_token, src, st);

  constexpr int DT = D / 32 / KH;                   // 32-element parts of a row that a wave ends up with
  if constexpr (KH == 2) add_halves<D, kFlWaves>(st, lds);
  const float l = sum_across32(st.l);
  const bool sees = lim >= 0;                       // else no key: zeros
  const float inv = 1.0f / l;
  uint16_t* op = a.out + (sr.q0 + static_cast<int64_t>(tok)) * a.o_token + hd * a.o_head + wave / RW * (D / 2);
  const bool live = wr0 + n < rows;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      // a lane half has elements 8 a + 4 hf .. +4 of a = 2c, 2c + 1: swapped, half hf has all 8 of a = 2c + hf
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = sees ? st.o[dt][8 * c + i] * inv : 0.0f;
      uint32_t lo[2], hi[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lo[i] = pack_bf16(y[2 * i], y[2 * i + 1]);
        hi[i] = pack_bf16(y[4 + 2 * i], y[4 + 2 * i + 1]);
      }
      const auto s0 = __builtin_amdgcn_permlane32_swap(lo[0], hi[0], false, false);
      const auto s1 = __builtin_amdgcn_permlane32_swap(lo[1], hi[1], false, false);
      if (live) *reinterpret_cast<u32x4*>(op + 32 * dt + 16 * c + 8 * hf) = u32x4{s0[0], s1[0], s0[1], s1[1]};
    }
}

}  // namespace

hipError_t launch_prompt(const dsk_prompt_desc& d, const void* q, const void* k, const void* v, const int32_t* cu_q,
                         const int32_t* cu_k, void* out, hipStream_t s) {
  const int group = d.heads / d.kv_heads;
  // every sequence's last tile may be partly filled
  auto blocks = [&](int rows) {
    return static_cast<unsigned>((static_cast<int64_t>(d.tokens) * group / rows + d.n_seqs) * d.kv_heads);
  };
  const PromptArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                     static_cast<uint16_t*>(out), cu_q, cu_k, d.q_token, d.q_head, d.k_token, d.k_head, d.v_token,
                     d.v_head, d.o_token, d.o_head, d.scale * kLog2e, d.tokens, d.kv_tokens, d.n_seqs, d.kv_heads,
                     group, d.causal, kCus / d.kv_heads};
  // Up to about one and a half workgroups a CU the time is that of the most keys, and two waves take
  // them for 32 rows (16 heads of 64 / 128: 2048 tokens 26.3 -> 21.5 / 35.9 -> 28.5 us, 32 rows
  // behind 8192 keys 81.5 -> 66.2 / 108 -> 71, prompts of 1500 and 1124 together 20.9 -> 17.6 / 29.6 -> 28.3, but
  // three of 1500 24.1 -> 27.7 / 38 -> 47), unless there are few (16 prompts of 128 tokens
  // 7.3 either way / 9.7 -> 11) or the loads of them, which are twice as many, bound it (64 times 32 rows
  // behind 2048 keys: 36 -> 48 / 62 -> 90)
  const bool few = static_cast<int64_t>(d.tokens) * group * d.kv_heads <= kCus * kFlRows * 3 / 2 &&
                   d.kv_tokens >= static_cast<int64_t>(d.n_seqs) * 4 * kFlKeys &&
                   static_cast<int64_t>(d.kv_tokens) * d.kv_heads * d.head_dim <= kFewElements;
  auto launch = [&](auto two, auto one, size_t lds) {
    if (few) launch_kernel(two, blocks(kFlRows / 2), kFlThreads, lds, s, a);
    else launch_kernel(one, blocks(kFlRows), kFlThreads, lds, s, a);
  };
  if (d.head_dim == 64) launch(k_prompt<64, 2>, k_prompt<64, 1>, flash_lds<64>());
  else launch(k_prompt<128, 2>, k_prompt<128, 1>, flash_lds<128>());
  return hipGetLastError();
}

}  // namespace dsk
