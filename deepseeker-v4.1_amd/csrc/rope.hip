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
// turn (error below 2^-50 position) goes to float32.  A block handles one token
// (or a part of its heads), so each pair's sine and cosine are computed once
// per token and shared through LDS.
#include "attn.h"

namespace dsk {
namespace {

constexpr int kQkThreads = 256;

struct QkArgs {
  const void *q, *k, *v;
  const int32_t *positions, *seq;
  const double* freq;
  const float *q_gamma, *k_gamma;
  uint16_t *q_out, *k_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, qo_token, qo_head, ko_token, ko_head;
  int32_t heads, kv_heads, rot_dim, rot_first, prefix_len, norm;
  float eps, mscale;
  CacheView cache;
  bool append;
};

template <bool kBF16>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&x)[8]) {
  if constexpr (kBF16) {
    const u32x4 r = ldg16(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(r[j] << 16);
      x[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
    }
  } else {
    const float* f = static_cast<const float*>(p) + i;
    const f32x4 a = ldg<f32x4>(f), b = ldg<f32x4>(f + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[j] = a[j]; x[4 + j] = b[j]; }
  }
}

__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r[j] = pack_bf16(x[2 * j], x[2 * j + 1]);
  return r;
}

// Rows of a token: its query heads, its key heads, and with a cache its value heads.
template <int D, bool kBF16, bool kInter>
__global__ __launch_bounds__(kQkThreads) void k_qk(const QkArgs a) {
  constexpr int kLanes = D / 8;                       // lanes of one head row
  constexpr int kRows = kQkThreads / kLanes;          // rows of one pass of the block
  __shared__ float2 turn[D / 2];
  const int64_t t = blockIdx.x;
  const int pos = a.positions[t];
  if (pos < 0) return;                                // a token of padding
  const int rows = a.heads + (a.append ? 2 : 1) * a.kv_heads;
  for (int i = threadIdx.x; i < a.rot_dim / 2; i += kQkThreads) {
    double r = static_cast<double>(pos) * (a.freq[i] * 0.15915494309189533577);   // turns: / (2 pi)
    r -= rint(r);
    float sn, cs;
    sincospif(2.0f * static_cast<float>(r), &sn, &cs);
    turn[i] = float2{cs * a.mscale, sn * a.mscale};
  }
  // the token's row of the cache, or none
  int64_t slot = -1;
  int in_page = 0;
  if (a.append) {
    const int s = a.seq[t];
    const int64_t at = static_cast<int64_t>(pos) - a.prefix_len;
    const int64_t page = at >> a.cache.page_shift;
    if (s >= 0 && s < a.cache.n_seqs && at >= 0 && page < a.cache.max_pages) {
      const int id = a.cache.table[s * a.cache.table_stride + page];
      if (id >= 0 && id < a.cache.n_pages) slot = id;
    }
    in_page = static_cast<int>(at & ((1 << a.cache.page_shift) - 1));
  }
  const int lane = threadIdx.x % kLanes, e = 8 * lane;
  const int half = a.rot_dim / 2, er = e - a.rot_first;       // this lane's first element among the rotated
  const bool rotated = er >= 0 && er < a.rot_dim;
  // half pairs: the elements that pair with the lane's own
  const int ep = kInter || !rotated ? e : (er < half ? e + half : e - half);
  bool first = true;
  for (int row = blockIdx.y * kRows + threadIdx.x / kLanes; row < rows || first; row += gridDim.y * kRows) {
    const int kind = row < a.heads ? 0 : row < a.heads + a.kv_heads ? 1 : 2;
    const int h = kind == 0 ? row : kind == 1 ? row - a.heads : row - a.heads - a.kv_heads;
    const bool live = row < rows;
    const void* src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const int64_t base = kind == 0   ? t * a.q_token + h * a.q_head
                         : kind == 1 ? t * a.k_token + h * a.k_head
                                     : t * a.v_token + h * a.v_head;
    float x[8], y[8];
    if (live) {
      load8<kBF16>(src, base + e, x);
      if (!kInter && kind != 2) load8<kBF16>(src, base + ep, y);
    }
    if (first) __syncthreads();                        // the turns are in LDS
    first = false;
    if (!live) break;
    if (kind != 2) {
      if (a.norm) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
        for (int m = kLanes / 2; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
        const float rstd = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
        const float* gamma = kind == 0 ? a.q_gamma : a.k_gamma;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = x[j] * rstd * (gamma ? gamma[e + j] : 1.0f);
          if (!kInter) y[j] = y[j] * rstd * (gamma ? gamma[ep + j] : 1.0f);
        }
      }
      if (rotated) {
        if constexpr (kInter) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 cs = turn[er / 2 + j];
            const float p = x[2 * j], q = x[2 * j + 1];
            x[2 * j] = p * cs.x - q * cs.y;
            x[2 * j + 1] = q * cs.x + p * cs.y;
          }
        } else {
          const float sign = er < half ? -1.0f : 1.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 cs = turn[(er < half ? er : er - half) + j];
            x[j] = x[j] * cs.x + sign * (y[j] * cs.y);
          }
        }
      }
    }
    const u32x4 r = pack8(x);
    if (kind == 0) {
      *reinterpret_cast<u32x4*>(a.q_out + t * a.qo_token + h * a.qo_head + e) = r;
    } else {
      if (kind == 1 && a.k_out) *reinterpret_cast<u32x4*>(a.k_out + t * a.ko_token + h * a.ko_head + e) = r;
      if (slot >= 0) {
        const int64_t at = (((slot * a.kv_heads + h) << a.cache.page_shift) + in_page) * D + e;
        *reinterpret_cast<u32x4*>((kind == 1 ? a.cache.k : a.cache.v) + at) = r;
      }
    }
  }
}

template <int D>
void launch_qk_d(const dsk_qk_desc& d, const QkArgs& a, hipStream_t s) {
  constexpr int kRows = kQkThreads / (D / 8);
  const int rows = d.heads + (a.append ? 2 : 1) * d.kv_heads;
  // few tokens: a token's heads over several blocks, so that one pass covers them
  const int passes = (rows + kRows - 1) / kRows;
  const dim3 grid(d.tokens, d.tokens < 512 ? passes : 1);
  if (d.dtype == DSK_DTYPE_BF16) {
    if (d.interleaved) launch_kernel(k_qk<D, true, true>, grid, kQkThreads, 0, s, a);
    else launch_kernel(k_qk<D, true, false>, grid, kQkThreads, 0, s, a);
  } else {
    if (d.interleaved) launch_kernel(k_qk<D, false, true>, grid, kQkThreads, 0, s, a);
    else launch_kernel(k_qk<D, false, false>, grid, kQkThreads, 0, s, a);
  }
}

}  // namespace

hipError_t launch_qk(const dsk_qk_desc& d, const void* q, const void* k, const void* v, const int32_t* positions,
                     const int32_t* seq, const double* freq, const float* q_gamma, const float* k_gamma,
                     const dsk_kv_cache* cache, void* q_out, void* k_out, hipStream_t s) {
  QkArgs a{q, k, v, positions, seq, freq, q_gamma, k_gamma, static_cast<uint16_t*>(q_out),
           static_cast<uint16_t*>(k_out), d.q_token, d.q_head, d.k_token, d.k_head, d.v_token, d.v_head,
           d.qo_token, d.qo_head, d.ko_token, d.ko_head, d.heads, d.kv_heads, d.rot_dim, d.rot_first,
           d.prefix_len, d.norm, d.eps, d.mscale, cache ? cache_view(*cache) : CacheView{}, cache != nullptr};
  if (d.head_dim == 64) launch_qk_d<64>(d, a, s);
  else launch_qk_d<128>(d, a, s);
  return hipGetLastError();
}

}  // namespace dsk
