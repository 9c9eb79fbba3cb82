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
  int32_t tokens, heads, kv_heads, rot_dim, rot_first, prefix_len, norm;
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

__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
}

// TB tokens a block; its rows are each token's query heads, its key heads, and
// with a cache its value heads.  A group of lanes takes one head of all TB tokens
// at a time, their loads together.
template <int D, bool kBF16, bool kInter, int TB>
__global__ __launch_bounds__(kQkThreads) void k_qk(const QkArgs a) {
  constexpr int kLanes = D / 8;                       // lanes of one head row
  constexpr int kRows = kQkThreads / kLanes;          // heads of one pass of the block
  __shared__ float2 turn[TB][D / 2];
  __shared__ __align__(16) float gam[2][D];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * TB;
  const int rows = a.heads + (a.append ? 2 : 1) * a.kv_heads;
  const int lane = threadIdx.x % kLanes, e = 8 * lane;
  const int half = a.rot_dim / 2, er = e - a.rot_first;       // this lane's first element among the rotated
  const bool rotated = er >= 0 && er < a.rot_dim;
  // half pairs: the elements that pair with the lane's own
  const int ep = kInter || !rotated ? e : (er < half ? e + half : e - half);

  int pos[TB];                                        // negative: padding
  int64_t slot[TB];                                   // the token's page, or -1
#pragma unroll
  for (int i = 0; i < TB; ++i) {
    pos[i] = t0 + i < a.tokens ? a.positions[t0 + i] : -1;
    slot[i] = -1;
    if (a.append && pos[i] >= 0) {
      const int s = a.seq[t0 + i];
      const int64_t at = static_cast<int64_t>(pos[i]) - a.prefix_len, page = at >> a.cache.page_shift;
      if (s >= 0 && s < a.cache.n_seqs && at >= 0 && page < a.cache.max_pages) {
        const int id = a.cache.table[s * a.cache.table_stride + page];
        if (id >= 0 && id < a.cache.n_pages) slot[i] = id;
      }
    }
  }
  auto source = [&](int row, int& kind, int& h, const void*& p, int64_t& token, int64_t& at) {
    kind = row < a.heads ? 0 : row < a.heads + a.kv_heads ? 1 : 2;
    h = kind == 0 ? row : kind == 1 ? row - a.heads : row - a.heads - a.kv_heads;
    p = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    token = kind == 0 ? a.q_token : kind == 1 ? a.k_token : a.v_token;
    at = t0 * token + h * (kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head);
  };
  Raw8<kBF16> x[TB], y[TB];
  auto load = [&](int row) {
    int kind, h;
    const void* p;
    int64_t token, at;
    source(row, kind, h, p, token, at);
#pragma unroll
    for (int i = 0; i < TB; ++i)
      if (pos[i] >= 0) {
        x[i].load(p, at + i * token + e);
        if (!kInter && kind != 2) y[i].load(p, at + i * token + ep);
      }
  };
  int row = blockIdx.y * kRows + threadIdx.x / kLanes;
  if (row < rows) load(row);                          // in flight while the angles are computed
  for (int i = threadIdx.x; i < TB * half; i += kQkThreads) {
    const int ti = i / half, pair = i - ti * half;
    const int p = t0 + ti < a.tokens ? a.positions[t0 + ti] : 0;
    double r = static_cast<double>(p) * (a.freq[pair] * 0.15915494309189533577);   // turns: / (2 pi)
    r -= rint(r);
    float sn, cs;
    sincospif(2.0f * static_cast<float>(r), &sn, &cs);
    turn[ti][pair] = float2{cs * a.mscale, sn * a.mscale};
  }
  for (int i = threadIdx.x; i < D; i += kQkThreads) {
    gam[0][i] = a.q_gamma ? a.q_gamma[i] : 1.0f;
    gam[1][i] = a.k_gamma ? a.k_gamma[i] : 1.0f;
  }
  __syncthreads();
  while (row < rows) {
    int kind, h;
    const void* p;
    int64_t token, at;
    source(row, kind, h, p, token, at);
    u32x4 out[TB];
#pragma unroll
    for (int i = 0; i < TB; ++i) {
      float z[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = x[i][j];
      if (kind != 2) {
        float rstd = 1.0f;
        if (a.norm) {
          float ss = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss += z[j] * z[j];
#pragma unroll
          for (int m = kLanes / 2; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
          rstd = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
        }
        const float* g = gam[kind];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = z[j] * rstd * g[e + j];
        if (rotated) {
          if constexpr (kInter) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 cs = turn[i][er / 2 + j];
              const float u = z[2 * j], v = z[2 * j + 1];
              z[2 * j] = u * cs.x - v * cs.y;
              z[2 * j + 1] = v * cs.x + u * cs.y;
            }
          } else {
            const float sign = er < half ? -rstd : rstd;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 cs = turn[i][(er < half ? er : er - half) + j];
              z[j] = z[j] * cs.x + (y[i][j] * sign * g[ep + j]) * cs.y;
            }
          }
        }
      }
      out[i] = pack8(z);
    }
    const int next = row + gridDim.y * kRows;
    // the next head's loads before this one's stores; results over the inputs stay
    // possible, since a head is read whole before its own stores
    if (next < rows) load(next);
#pragma unroll
    for (int i = 0; i < TB; ++i) {
      if (pos[i] < 0) continue;
      const int64_t t = t0 + i;
      if (kind == 0) {
        *reinterpret_cast<u32x4*>(a.q_out + t * a.qo_token + h * a.qo_head + e) = out[i];
      } else {
        if (kind == 1 && a.k_out) *reinterpret_cast<u32x4*>(a.k_out + t * a.ko_token + h * a.ko_head + e) = out[i];
        if (slot[i] >= 0) {
          const int in_page = static_cast<int>((pos[i] - a.prefix_len) & ((1 << a.cache.page_shift) - 1));
          const int64_t to = (((slot[i] * a.kv_heads + h) << a.cache.page_shift) + in_page) * D + e;
          *reinterpret_cast<u32x4*>((kind == 1 ? a.cache.k : a.cache.v) + to) = out[i];
        }
      }
    }
    row = next;
  }
}

template <int D, int TB>
void launch_qk_t(const dsk_qk_desc& d, const QkArgs& a, dim3 grid, hipStream_t s) {
  if (d.dtype == DSK_DTYPE_BF16) {
    if (d.interleaved) launch_kernel(k_qk<D, true, true, TB>, grid, kQkThreads, 0, s, a);
    else launch_kernel(k_qk<D, true, false, TB>, grid, kQkThreads, 0, s, a);
  } else {
    if (d.interleaved) launch_kernel(k_qk<D, false, true, TB>, grid, kQkThreads, 0, s, a);
    else launch_kernel(k_qk<D, false, false, TB>, grid, kQkThreads, 0, s, a);
  }
}

template <int D>
void launch_qk_d(const dsk_qk_desc& d, const QkArgs& a, hipStream_t s) {
  constexpr int kRows = kQkThreads / (D / 8);
  const int rows = d.heads + (a.append ? 2 : 1) * d.kv_heads;
  const int passes = (rows + kRows - 1) / kRows;
  // few tokens: one a block, its heads over several blocks, so that one pass covers them
  if (d.tokens < 1024) launch_qk_t<D, 1>(d, a, dim3(d.tokens, passes), s);
  else launch_qk_t<D, 4>(d, a, dim3((d.tokens + 3) / 4, 1), s);
}

}  // namespace

hipError_t launch_qk(const dsk_qk_desc& d, const void* q, const void* k, const void* v, const int32_t* positions,
                     const int32_t* seq, const double* freq, const float* q_gamma, const float* k_gamma,
                     const CacheView* cache, void* q_out, void* k_out, hipStream_t s) {
  QkArgs a{q, k, v, positions, seq, freq, q_gamma, k_gamma, static_cast<uint16_t*>(q_out),
           static_cast<uint16_t*>(k_out), d.q_token, d.q_head, d.k_token, d.k_head, d.v_token, d.v_head,
           d.qo_token, d.qo_head, d.ko_token, d.ko_head, d.tokens, d.heads, d.kv_heads, d.rot_dim, d.rot_first,
           d.prefix_len, d.norm, d.eps, d.mscale, cache ? *cache : CacheView{}, cache != nullptr};
  if (d.head_dim == 64) launch_qk_d<64>(d, a, s);
  else launch_qk_d<128>(d, a, s);
  return hipGetLastError();
}

}  // namespace dsk
