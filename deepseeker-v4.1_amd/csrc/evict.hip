// Eviction from a paged cache: of every sequence longer than `keep`, each key head keeps
// its first `first` rows, its last `recent` ones, and of the others those of most accumulated
// weight (of equal ones the first), in the rows 0 .. keep - 1.
//
// As few rows move as can: with middle = keep - recent, kept rows in front of it stay, the i-th kept row
// behind it that is not one of the last goes to the i-th row there that is given up (a hole), and the last
// rows follow in their order.  Every row comes from one at least as far behind, src[j] >= j.
//
// Two kernels.  k_evict_pick, a workgroup for a (sequence, head): the m-th largest weight by its bits, 8 at
// a time, from counts in LDS; then the lists of holes and of rows that fill them: 12.6 us for 512 times 1088
// weights, 16.3 for 32 times up to 16000, nearly all of it passes over LDS and their barriers.  k_evict_move copies:
// what comes from behind the first `keep` rows is written nowhere, so workgroups share it freely; what comes
// from within them, and the last rows, whose places may overlap, one workgroup moves in order, a piece
// read whole before it is written.  24.4 us for 98 MB read and written (4.0 TB/s; a large copy 4.9).
//
// In 8 bits a block of 16 rows has one scale: a block with a row from elsewhere takes the largest of its rows'
// scales, and its rows move to it, so blocks are made whole.  Rows behind the kept ones in the last block do not: they are none of the
// sequence's any more, and a smaller scale might not hold them.
#include <algorithm>

#include "kv8.h"

namespace dsk {
namespace {

constexpr int kMoveThreads = 1024;

// A block with holes (one bit each of mask), which are filled from fills[start ..].
struct EvictBlock { int32_t block, start; uint32_t mask; int32_t unused; };
// Of an item: its holes; those that rows fill which a move may write; blocks with holes.
struct EvictCounts { int32_t holes, near, blocks, unused; };

struct EvictArgs {
  CacheView c;
  uint8_t *k_scale, *v_scale;
  float* weights;
  const int32_t* lens;
  int32_t* lens_out;
  int32_t *holes, *fills;            // [item][most]: rows that are filled, and whence
  EvictBlock* blocks;                // [item][most], of a cache in 8 bits
  EvictCounts* counts;               // [item]
  int64_t most;
  int32_t kv_heads, keep, first, recent, slices;
};

// Rows of sequence b, or 0 where there is nothing to do: `keep` or fewer, or more than the table row holds.
__device__ __forceinline__ int rows_of(const EvictArgs& a, int b) {
  const int n = a.lens[b];
  return n <= a.keep || n > static_cast<int64_t>(a.c.max_pages) << a.c.page_shift ? 0 : n;
}

// Row of the cache (of one head of a page) that row j of sequence b is, or -1: on a page outside the cache.
__device__ __forceinline__ int64_t cache_row(const EvictArgs& a, int b, int h, int j) {
  const int id = ldg<int32_t>(a.c.table + b * a.c.table_stride + (j >> a.c.page_shift));
  if (id < 0 || id >= a.c.n_pages) return -1;
  return ((static_cast<int64_t>(id) * a.kv_heads + h) << a.c.page_shift) + (j & ((1 << a.c.page_shift) - 1));
}

// Order of weights as unsigned numbers: NaN above all, -0 as 0; a row on a page outside the cache below.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  if (w != w) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

typedef f32x4 f32x4_a4 __attribute__((aligned(4)));   // weights may start anywhere

// Sum of v over the threads before this one, and over all; `waves`: LDS for a number of each wave.
template <int kWaves>
__device__ __forceinline__ uint32_t before_me(uint32_t v, uint32_t& all, uint32_t* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t up = v;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t x = __shfl_up(up, s, 64);
    if (lane >= s) up += x;
  }
  if (lane == 63) waves[wave] = up;
  __syncthreads();
  uint32_t before = up - v;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint32_t n = waves[w];
    if (w < wave) before += n;
    all += n;
  }
  return before;
}

// A thread takes 16 rows one after the other: they lie in one page, and what becomes of them is a mask (that of
// the block's holes, in 8 bits); sums over threads are two scans.  Kept in registers, so that a workgroup reads up to 16
// kThreads rows once.  (A row a thread in rounds, with a ballot and a sum for each: 61 us for 16000 rows and 16 for 1088.)
template <int kThreads>
__global__ __launch_bounds__(kThreads) void k_evict_pick(const EvictArgs a) {
  constexpr int kWaves = kThreads / 64, kRows = kScaleRows * kThreads, kCopies = 4;
  __shared__ uint32_t counts[kCopies][256 + 8];       // of digits: lanes of the same one meet less often in four
  __shared__ uint32_t chosen[3];                      // digit, rows above it, rows that have it
  __shared__ uint32_t sums[3][kWaves];
  const int item = blockIdx.x, b = item / a.kv_heads, h = item % a.kv_heads, tid = threadIdx.x;
  const int n = rows_of(a, b);
  if (h == 0 && tid == 0 && a.lens_out != a.lens) a.lens_out[b] = n ? a.keep : a.lens[b];
  if (n == 0) return;                                 // (the moves do not look either)
  const int from = a.first, to = n - a.recent;        // the free rows
  const int want = a.keep - a.first - a.recent;       // how many of them stay: fewer than there are
  const int base0 = from / kScaleRows * kScaleRows;
  uint32_t key[kScaleRows], is_free = 0;              // of the rows from `row0` on; a bit a row
  int held = -1, row0 = 0;
  auto hold = [&](int base) {
    if (held == base) return;
    held = base;
    row0 = base + tid * kScaleRows;
    is_free = 0;
    if (row0 >= to) return;
    is_free = 0xffffu;
    if (row0 < from) is_free &= 0xffffu << (from - row0);
    if (to - row0 < kScaleRows) is_free &= (1u << (to - row0)) - 1;
    const int64_t row = cache_row(a, b, h, row0);
#pragma unroll
    for (int i = 0; i < kScaleRows; i += 4) {
      const f32x4 w = row < 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const f32x4_a4*>(a.weights + row + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) key[i + j] = row < 0 ? 0 : order_of(w[j]);
    }
  };
  // the want-th largest key: the digits from `shift` on known, `left` rows to find among those that share them
  uint32_t cut = 0;
  int left = want;
  for (int shift = 24; left > 0 && shift >= 0; shift -= 8) {
    for (int i = tid; i < kCopies * (256 + 8); i += kThreads) (&counts[0][0])[i] = 0;
    __syncthreads();
    for (int base = base0; base < to; base += kRows) {
      hold(base);
#pragma unroll
      for (int i = 0; i < kScaleRows; ++i)
        if ((is_free >> i & 1) && (shift == 24 || (key[i] ^ cut) >> (shift + 8) == 0))
          atomicAdd(&counts[tid & (kCopies - 1)][key[i] >> shift & 255], 1u);
    }
    __syncthreads();
    if (tid < 64) {                                   // lane i: digits 255 - 4 i and the three below
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = 0;
#pragma unroll
        for (int k = 0; k < kCopies; ++k) c[i] += counts[k][255 - 4 * tid - i];
        sum += c[i];
      }
      uint32_t up = sum;
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) {
        const uint32_t v = __shfl_up(up, s, 64);
        if (tid >= s) up += v;
      }
      uint32_t above = up - sum;                      // rows with larger digits
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < static_cast<uint32_t>(left) && above + c[i] >= static_cast<uint32_t>(left)) {
          chosen[0] = 255 - 4 * tid - i;
          chosen[1] = above;
          chosen[2] = c[i];
        }
        above += c[i];
      }
    }
    __syncthreads();
    cut |= chosen[0] << shift;
    left -= static_cast<int>(chosen[1]);
    if (static_cast<int>(chosen[2]) == left && cut != 0) {   // all rows with these digits stay: no need for the others
      --cut;
      left = 0;
    }
  }
  // rows above the cut stay, and the first `left` of those at it
  int32_t *holes = a.holes + item * a.most, *fills = a.fills + item * a.most;
  EvictBlock* list = a.blocks + item * a.most;
  const int middle = a.keep - a.recent;
  const int bound = a.k_scale ? (a.keep + kScaleRows - 1) / kScaleRows * kScaleRows : a.keep;   // rows that a move may write
  int equal = 0, hole = 0, fill = 0, near = 0, blocks = 0;
  for (int base = base0; base < to; base += kRows) {
    hold(base);
    uint32_t stay = 0, ties = 0;
    if (is_free) {
#pragma unroll
      for (int i = 0; i < kScaleRows; ++i) {
        stay |= key[i] > cut ? 1u << i : 0;
        ties |= key[i] == cut ? 1u << i : 0;
      }
      stay = want > 0 ? stay & is_free : 0;
      ties &= is_free;
    }
    if (left > 0) {
      uint32_t all;
      int before = equal + static_cast<int>(before_me<kWaves>(__popc(ties), all, sums[0]));
      equal += static_cast<int>(all);
      for (; ties && before < left; ++before, ties &= ties - 1) stay |= ties & -ties;
    }
    // rows in front of middle, and of `bound`, in this thread's block
    auto up_to = [&](int end) { return end <= row0 ? 0u : end - row0 >= kScaleRows ? 0xffffu : (1u << (end - row0)) - 1; };
    const uint32_t front = up_to(middle), gone = is_free & front & ~stay, come = stay & ~front;
    uint32_t all, others;
    const uint32_t before = before_me<kWaves>(__popc(gone) | __popc(come) << 16, all, sums[1]);
    const uint32_t more = before_me<kWaves>((gone ? 1 : 0) | __popc(come & up_to(bound)) << 16, others, sums[2]);
    int at_hole = hole + static_cast<int>(before & 0xffff), at_fill = fill + static_cast<int>(before >> 16);
    if (a.k_scale) {
      const int at = blocks + static_cast<int>(more & 0xffff);
      if (gone && at < a.most) list[at] = EvictBlock{row0 / kScaleRows, at_hole, gone, 0};
    } else {
      for (uint32_t m = gone; m; m &= m - 1, ++at_hole)
        if (at_hole < a.most) holes[at_hole] = row0 + __ffs(static_cast<int>(m)) - 1;
    }
    for (uint32_t m = come; m; m &= m - 1, ++at_fill)
      if (at_fill < a.most) fills[at_fill] = row0 + __ffs(static_cast<int>(m)) - 1;
    hole += static_cast<int>(all & 0xffff);
    fill += static_cast<int>(all >> 16);
    blocks += static_cast<int>(others & 0xffff);
    near += static_cast<int>(others >> 16);
    __syncthreads();                                  // sums have been read
  }
  if (tid == 0) a.counts[item] = EvictCounts{hole, near, blocks, 0};
}

// bf16: pieces of 16 bytes, K and V of a row after each other; the weight with the first.
template <int D>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int b, int h, int n, const int32_t* holes, const int32_t* fills,
                                          int i0, int i1, bool window) {
  constexpr int kPieces = 2 * D / 8, kAhead = 8;
  const int middle = a.keep - a.recent, d = n - a.keep;
  // move m of i1 - i0 fills, then of the last rows
  const int64_t all = static_cast<int64_t>(i1 - i0 + (window ? a.recent : 0)) * kPieces;
  for (int64_t p0 = 0; p0 < all; p0 += kAhead * kMoveThreads) {
    u32x4 x[kAhead];
    float w[kAhead];
    int64_t to[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t p = p0 + i * kMoveThreads + threadIdx.x;
      to[i] = -1;
      if (p >= all) continue;
      const int m = static_cast<int>(p / kPieces) + i0, piece = static_cast<int>(p % kPieces);
      const int dst = m < i1 ? holes[m] : middle + m - i1, src = m < i1 ? fills[m] : dst + d;
      const int64_t r = cache_row(a, b, h, src);
      if (r < 0) continue;
      to[i] = cache_row(a, b, h, dst);
      x[i] = ldg16((piece < D / 8 ? a.c.k : a.c.v) + r * D + 8 * (piece % (D / 8)));
      if (piece == 0) w[i] = ldg<float>(a.weights + r);
    }
    if (window) __syncthreads();                      // read whole before it is written
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int piece = static_cast<int>((p0 + i * kMoveThreads + threadIdx.x) % kPieces);
      if (to[i] < 0) continue;
      *reinterpret_cast<u32x4*>((piece < D / 8 ? a.c.k : a.c.v) + to[i] * D + 8 * (piece % (D / 8))) = x[i];
      if (piece == 0) a.weights[to[i]] = w[i];
    }
  }
}

template <int D>
__global__ __launch_bounds__(kMoveThreads) void k_evict_move(const EvictArgs a) {
  const int item = blockIdx.x / a.slices, slice = blockIdx.x % a.slices, b = item / a.kv_heads, h = item % a.kv_heads;
  const int n = rows_of(a, b);
  if (n == 0) return;
  const EvictCounts count = a.counts[item];
  const int32_t *holes = a.holes + item * a.most, *fills = a.fills + item * a.most;
  // slice 0: what comes from the first rows, then the last rows; all: their share of the others
  const int64_t free = count.holes - count.near;
  const int i0 = slice ? count.near + static_cast<int>(free * slice / a.slices) : 0;
  const int i1 = count.near + static_cast<int>(free * (slice + 1) / a.slices);
  move_rows<D>(a, b, h, n, holes, fills, i0, i1, slice == 0);
}

// In 8 bits, by blocks: a wave takes a block's 16 rows of K or of V, four lanes a row, so that their largest scale stays
// in the wave.
template <int D>
struct CodeBlock {
  static constexpr int kPieces = D / 64;              // 16 bytes each, of a lane
  u32x4 x[kPieces];
  int64_t from, to;                                   // the lane's row: whence, and whereto (-1: nowhere)
  uint32_t byte;
  float weight;

  // mask: the rows that are holes, filled from fills[0 ..]; from row `middle` on: from d rows behind
  __device__ __forceinline__ void load(const EvictArgs& a, int b, int h, int block, uint32_t mask, const int32_t* fills, int middle,
                                       int d, int w) {
    const int lane = threadIdx.x & 63, r = lane >> 2, part = lane & 3, j = block * kScaleRows + r;
    to = from = -1;
    byte = 0;
    if (j >= a.keep) return;
    int src = j;
    if (j >= middle) src = j + d;
    else if (mask >> r & 1) src = fills[__popc(mask & ((1u << r) - 1))];
    to = cache_row(a, b, h, j);
    if (to < 0) return;
    from = cache_row(a, b, h, src);
    if (from < 0) from = to;                          // no such row: the one there stays
    const uint8_t* p = reinterpret_cast<const uint8_t*>(w ? a.c.v : a.c.k) + from * D + part * (D / 4);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) x[i] = ldg16(p + 16 * i);
    byte = ldg<uint8_t>((w ? a.v_scale : a.k_scale) + from / kScaleRows);
    if (w == 0 && part == 0) weight = ldg<float>(a.weights + from);
  }
  __device__ __forceinline__ void store(const EvictArgs& a, int w) {
    const int lane = threadIdx.x & 63, part = lane & 3;
    uint32_t top = byte;
#pragma unroll
    for (int s = 4; s < 64; s <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), s, 64)));
    if (to < 0) return;
    const float f = scale_step(static_cast<int>(byte), static_cast<int>(top));
    if (byte != top)
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) x[i][k] = rescale4(x[i][k], f);
    uint8_t* p = reinterpret_cast<uint8_t*>(w ? a.c.v : a.c.k) + to * D + part * (D / 4);
    if (from != to || byte != top)
#pragma unroll
      for (int i = 0; i < kPieces; ++i) *reinterpret_cast<u32x4*>(p + 16 * i) = x[i];
    if (lane == 0) (w ? a.v_scale : a.k_scale)[to / kScaleRows] = static_cast<uint8_t>(top);
    if (w == 0 && part == 0 && from != to) a.weights[to] = weight;
  }
};

template <int D>
__global__ __launch_bounds__(kMoveThreads) void k_evict_move_codes(const EvictArgs a) {
  constexpr int kAhead = 4, kPairs = kMoveThreads / 128;   // of waves, a block each
  __shared__ int n_near;
  const int item = blockIdx.x / a.slices, slice = blockIdx.x % a.slices, b = item / a.kv_heads, h = item % a.kv_heads;
  const int n = rows_of(a, b);
  if (n == 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pair = wave >> 1, w = wave & 1;
  const EvictCounts count = a.counts[item];
  const int32_t* fills = a.fills + item * a.most;
  const EvictBlock* list = a.blocks + item * a.most;
  const int middle = a.keep - a.recent, d = n - a.keep, blocks = (a.keep + kScaleRows - 1) / kScaleRows;
  // the first block with one of the last rows, or with a row behind those that are kept: its scale is read
  // for rows behind `middle` as well as written, in order
  const int window = middle / kScaleRows;
  // (the list's last block may be that one)
  const bool both = count.blocks > 0 && list[count.blocks - 1].block == window;
  const int listed = count.blocks - (both ? 1 : 0);
  // blocks with a row from those that the window's moves write are slice 0's
  if (threadIdx.x == 0) n_near = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < min(listed, count.near); i += kMoveThreads)
    if (list[i].start < count.near) atomicAdd(&n_near, 1);
  __syncthreads();
  const int near = n_near;
  auto some = [&](int i0, int i1) {
    for (int i = i0 + pair; i < i1; i += kAhead * kPairs) {
      CodeBlock<D> x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u * kPairs < i1) {
          const EvictBlock e = list[i + u * kPairs];
          x[u].load(a, b, h, e.block, e.mask, fills + e.start, middle, d, w);
        }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u * kPairs < i1) x[u].store(a, w);
    }
  };
  const int64_t free = listed - near;
  some(slice ? near + static_cast<int>(free * slice / a.slices) : 0, near + static_cast<int>(free * (slice + 1) / a.slices));
  if (slice) return;
  __syncthreads();                                    // their reads, before the window's writes
  for (int i0 = window; i0 < blocks; i0 += kAhead * kPairs) {
    CodeBlock<D> x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int block = i0 + u * kPairs + pair;
      const bool first = both && block == window;
      if (block < blocks)
        x[u].load(a, b, h, block, first ? list[listed].mask : 0u, first ? fills + list[listed].start : fills, middle, d, w);
    }
    __syncthreads();                                  // read whole before it is written
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i0 + u * kPairs + pair < blocks) x[u].store(a, w);
  }
}

__global__ void k_evict_lens(int32_t* lens, int batch, int keep, int64_t cap) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < batch && lens[b] > keep && lens[b] <= cap) lens[b] = keep;
}

struct EvictPlan {
  int64_t most;
  size_t holes, fills, blocks, counts, total;
};

EvictPlan plan_of(const dsk_evict_desc& d, const dsk_kv_cache& c, bool codes) {
  EvictPlan p{};
  auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
  const int64_t items = static_cast<int64_t>(c.n_seqs) * d.kv_heads, cap = static_cast<int64_t>(c.max_pages) * c.page_size;
  // holes are among the rows that are given up, and each takes one of those that stay
  p.most = std::max<int64_t>(std::min<int64_t>(d.keep - d.first - d.recent, cap - d.keep), 1);
  p.holes = 0;
  p.fills = codes ? 0 : up(static_cast<size_t>(items * p.most) * 4);
  p.blocks = p.fills + up(static_cast<size_t>(items * p.most) * 4);
  p.counts = p.blocks + (codes ? up(static_cast<size_t>(items * p.most) * sizeof(EvictBlock)) : 0);
  p.total = p.counts + up(static_cast<size_t>(items) * sizeof(EvictCounts));
  return p;
}

// Workgroups of the moves, at least about.
constexpr int kMoveBlocks = 512, kMostSlices = 16;

template <int D>
void launch_evict_d(const EvictArgs& a, int items, hipStream_t s) {
  // a table row that 256 threads hold at once needs no more
  if ((static_cast<int64_t>(a.c.max_pages) << a.c.page_shift) <= 256 * kScaleRows) launch_kernel(k_evict_pick<256>, items, 256, 0, s, a);
  else launch_kernel(k_evict_pick<1024>, items, 1024, 0, s, a);
  launch_kernel(a.k_scale ? k_evict_move_codes<D> : k_evict_move<D>, items * a.slices, kMoveThreads, 0, s, a);
}

}  // namespace

size_t evict_workspace(const dsk_evict_desc& d, const dsk_kv_cache& c, bool codes) { return plan_of(d, c, codes).total; }

hipError_t launch_evict(const dsk_evict_desc& d, const dsk_kv_cache& c, const CacheView& view, uint8_t* k_scale, uint8_t* v_scale,
                        float* weights, const int32_t* lens, int32_t* lens_out, void* ws, hipStream_t s) {
  const EvictPlan p = plan_of(d, c, k_scale != nullptr);
  char* w = static_cast<char*>(ws);
  const int items = c.n_seqs * d.kv_heads;
  const int slices = std::min(std::max(kMoveBlocks / items, 1), kMostSlices);
  const EvictArgs a{view, k_scale, v_scale, weights, lens, lens_out, reinterpret_cast<int32_t*>(w + p.holes),
                    reinterpret_cast<int32_t*>(w + p.fills), reinterpret_cast<EvictBlock*>(w + p.blocks),
                    reinterpret_cast<EvictCounts*>(w + p.counts), p.most, d.kv_heads, d.keep, d.first, d.recent, slices};
  if (d.head_dim == 64) launch_evict_d<64>(a, items, s);
  else launch_evict_d<128>(a, items, s);
  if (lens_out == lens)
    launch_kernel(k_evict_lens, (c.n_seqs + 255) / 256, 256, 0, s, lens_out, c.n_seqs, d.keep, static_cast<int64_t>(c.max_pages) * c.page_size);
  return hipGetLastError();
}

}  // namespace dsk
