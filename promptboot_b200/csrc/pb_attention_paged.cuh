// Work division of the paged serving attention, shared by its kernels.
//
// Rows are packed: the rows of one (sequence, key head) are its tokens or nodes
// times the query heads that share the key head, row r = token * group + head, so
// that grouped heads and short sequences fill a row tile.  A row tile of one
// (sequence, key head) is a segment; its keys are walked in tiles.
//
// Prompts: one CTA per segment, the row tiles of a sequence from its end (the
// longest) to its start.  Trees: all key tiles of all segments form one list,
// which the CTAs share out evenly in consecutive runs whatever the sequences'
// lengths are; a segment that crosses runs leaves one partial (weighted sum,
// maximum, sum) per run in the workspace and combine_kernel joins them.
#pragma once

#include "pb_common.cuh"
#include "pb_kernels.cuh"
#include "pb_paged.cuh"

#include <algorithm>

namespace pb {
namespace paged {

struct AttnArgs {
  pb_rows q, k, v, out;  // k, v: packed keys (prompts)
  CacheView cache;       // trees
  const uint32_t* q_offsets;
  const uint32_t* kv_offsets;  // prompts
  const uint32_t* tables;      // trees, with contexts and visible
  const uint32_t* contexts;
  const unsigned long long* visible;
  uint32_t seqs, q_rows, kv_rows, kv_heads, group, table_width;
  float scale_log2;  // scale * log2(e): weights are powers of two
  float* partial;
};

// One sequence: its rows of q, its keys, and how many of them every row sees.
struct Sequence {
  uint32_t q0, t;     // first q row, tokens or nodes
  uint32_t kv0, len;  // first packed key (prompts), keys
  uint32_t context;   // trees
};

template <bool kTree>
__device__ __forceinline__ Sequence load_sequence(const AttnArgs& a, uint32_t s) {
  Sequence q;
  q.q0 = min(a.q_offsets[s], a.q_rows);
  const uint32_t q1 = min(a.q_offsets[s + 1], a.q_rows);
  q.t = q1 > q.q0 ? q1 - q.q0 : 0;
  if (kTree) {
    const uint32_t reach = a.table_width * a.cache.page_size;
    q.kv0 = 0;
    q.context = min(a.contexts[s], reach);
    q.len = min(q.context + min(q.t, 64u), reach);
  } else {
    q.kv0 = min(a.kv_offsets[s], a.kv_rows);
    const uint32_t k1 = min(a.kv_offsets[s + 1], a.kv_rows);
    q.len = k1 > q.kv0 ? k1 - q.kv0 : 0;
    q.context = 0;
  }
  return q;
}

// What one row sees: every key below `all` and the keys all + b of the set bits b.
struct RowView {
  uint32_t all;
  unsigned long long bits;
  __device__ __forceinline__ bool sees(uint32_t key) const {
    return key < all || (key - all < 64u && ((bits >> (key - all)) & 1ull));
  }
};
template <bool kTree>
__device__ __forceinline__ RowView row_view(const AttnArgs& a, const Sequence& s, uint32_t token) {
  if (kTree) {
    const uint32_t nodes = s.len - s.context;
    unsigned long long bits = a.visible[s.q0 + token];
    if (nodes < 64) bits &= (1ull << nodes) - 1ull;
    return {s.context, bits};
  }
  const uint32_t seen = s.len + token + 1;
  return {seen > s.t ? seen - s.t : 0, 0ull};
}

__device__ __forceinline__ uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

// Segments (prompts) or key tiles (trees) of a sequence, per key head and in all.
template <bool kTree, int kRows, int kKeys>
__device__ __forceinline__ uint32_t sequence_work(const AttnArgs& a, const Sequence& s) {
  const uint32_t segments = ceil_div(s.t * a.group, kRows) * a.kv_heads;
  return kTree ? segments * max(1u, ceil_div(s.len, kKeys)) : segments;
}

// Inclusive prefix of the sequences' work in shared memory; every thread of the
// block calls it.  A thread takes consecutive sequences, so that one scan of the block
// serves them all.  seqs <= PB_MAX_SEQS.
template <bool kTree, int kRows, int kKeys, int kThreads>
__device__ __forceinline__ void work_prefix(const AttnArgs& a, uint32_t* prefix) {
  __shared__ uint32_t warp_sum[kThreads / 32];
  const uint32_t each = ceil_div(a.seqs, kThreads), first = threadIdx.x * each;
  const uint32_t last = min(a.seqs, first + each);
  uint32_t sum = 0;
#pragma unroll 4
  for (uint32_t s = first; s < last; ++s) {
    sum += sequence_work<kTree, kRows, kKeys>(a, load_sequence<kTree>(a, s));
    prefix[s] = sum;
  }
  uint32_t scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, scan, d);
    if ((threadIdx.x & 31) >= d) scan += o;
  }
  if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x >> 5] = scan;
  __syncthreads();
  uint32_t before = scan - sum;
  for (int i = 0; i < (int)(threadIdx.x >> 5); ++i) before += warp_sum[i];
  if (before)
    for (uint32_t s = first; s < last; ++s) prefix[s] += before;
  __syncthreads();
}

// The sequence that holds item x of the prefix, and x within it.
__device__ __forceinline__ uint32_t find_sequence(const uint32_t* prefix, uint32_t seqs, uint32_t& x) {
  uint32_t lo = 0, hi = seqs - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) >> 1;
    if (x < prefix[mid]) hi = mid;
    else lo = mid + 1;
  }
  if (lo) x -= prefix[lo - 1];
  return lo;
}

// The trees' list of `total` key tiles over `grid` CTAs, at least kLeast tiles
// each: CTA c takes [start(c), start(c + 1)), and tile x belongs to CTA holder(x).
template <int kLeast>
struct Share {
  uint32_t total, ctas;
  __device__ __forceinline__ Share(uint32_t total_, uint32_t grid)
      : total(total_), ctas(min(grid, max(1u, total_ / kLeast))) {}
  __device__ __forceinline__ uint32_t start(uint32_t c) const {
    return (uint32_t)((uint64_t)c * total / ctas);
  }
  __device__ __forceinline__ uint32_t holder(uint32_t x) const {
    return (uint32_t)((((uint64_t)x + 1) * ctas - 1) / total);
  }
};

// A run of key tiles [tile0, tile1) of one segment.
struct Piece {
  uint32_t seq, head, row_tile;
  uint32_t tile0, tile1;
  int partial;  // workspace record, -1: the whole segment, straight to out
};

// Takes the next piece of a CTA's items [next, end).
template <bool kTree, int kRows, int kKeys>
__device__ __forceinline__ void take_piece(const AttnArgs& a, const uint32_t* prefix, uint32_t& next, uint32_t end,
                                           Piece& p, Sequence& s, uint32_t& rows) {
  uint32_t x = next;
  p.seq = find_sequence(prefix, a.seqs, x);
  s = load_sequence<kTree>(a, p.seq);
  rows = s.t * a.group;
  const uint32_t row_tiles = ceil_div(rows, kRows);
  p.partial = -1;
  if (kTree) {
    const uint32_t tiles = max(1u, ceil_div(s.len, kKeys));
    p.tile0 = x % tiles;
    p.tile1 = min(tiles, p.tile0 + (end - next));
    p.head = x / tiles / row_tiles;
    p.row_tile = x / tiles % row_tiles;
    if (p.tile0 > 0 || p.tile1 < tiles) p.partial = (int)(2 * blockIdx.x + (p.tile0 == 0));
    next += p.tile1 - p.tile0;
    if (s.len == 0) p.tile1 = p.tile0 = 0;  // nothing to see
  } else {
    p.head = x % a.kv_heads;
    p.row_tile = row_tiles - 1 - x / a.kv_heads;
    const uint32_t last = min(rows, (p.row_tile + 1) * kRows) - 1;
    p.tile0 = 0;
    p.tile1 = ceil_div(row_view<false>(a, s, last / a.group).all, kKeys);
    ++next;
  }
}

// The partial of CTA c for a segment that began before it, or that begins in it.
__device__ __forceinline__ int partial_of(uint32_t cta, bool begins) { return (int)(2 * cta + begins); }

// Four consecutive elements, rounded once.
__device__ __forceinline__ void store4(float* out, float4 y) { *reinterpret_cast<float4*>(out) = y; }
template <class T>
__device__ __forceinline__ void store4(T* out, float4 y) {
  *reinterpret_cast<uint2*>(out) =
      make_uint2(Elements<T>::pair(y.x, y.y), Elements<T>::pair(y.z, y.w));
}

template <int kRows, int kDim>
__host__ __device__ constexpr size_t partial_words() {
  return (size_t)kRows * (kDim + 2);
}

// Joins the partials of the segments that crossed CTA runs: weights 2^(m_i - m),
// in the order of the runs, so the result does not depend on timing.  A segment
// is joined by the CTAs (four at most, so that one wave of them holds all) of the edge
// at the end of the run in which it begins.  A thread has four elements of a row and
// loads eight partials at a time: latency is what there is to save here.
template <class T, int kDim, int kRows, int kKeys, int kLeast>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ AttnArgs a, uint32_t grid) {
  extern __shared__ uint32_t prefix[];
  work_prefix<true, kRows, kKeys, 256>(a, prefix);
  const uint32_t total = prefix[a.seqs - 1], c = blockIdx.x;
  const Share<kLeast> share(max(1u, total), grid);
  bool mine = total > 0 && c + 1 < share.ctas;
  uint32_t edge = 0, begin = 0, seq = 0, x = 0, tiles = 1;
  Sequence s{};
  if (mine) {
    x = edge = share.start(c + 1);
    seq = find_sequence(prefix, a.seqs, x);
    s = load_sequence<true>(a, seq);
    tiles = max(1u, ceil_div(s.len, kKeys));
    begin = edge - x % tiles;
    mine = begin != edge && begin >= share.start(c);  // else it begins at the edge, or in an earlier run
  }
  pdl_wait();  // the partials; also in a CTA that has none, for what comes after this launch
  if (!mine) return;
  constexpr int kPerRow = kDim / 4, kStep = 256 / kPerRow, kBatch = 8;
  const uint32_t last = share.holder(begin + tiles - 1);
  const uint32_t row_tiles = ceil_div(s.t * a.group, kRows);
  const uint32_t head = x / tiles / row_tiles, row_tile = x / tiles % row_tiles;
  const int chunk = (threadIdx.x % kPerRow) * 4;
  for (uint32_t r = blockIdx.y * kStep + threadIdx.x / kPerRow; r < kRows; r += gridDim.y * kStep) {
    const uint32_t row = row_tile * kRows + r;
    if (row >= s.t * a.group) return;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t p0 = c; p0 <= last; p0 += kBatch) {
      float mp[kBatch], lp[kBatch];
      float4 op[kBatch];
      float to = m;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        mp[i] = -INFINITY;
        if (p0 + i <= last) {
          const float* rec = a.partial + partial_of(p0 + i, p0 + i == c) * partial_words<kRows, kDim>();
          mp[i] = rec[kRows * kDim + r];
          lp[i] = rec[kRows * kDim + kRows + r];
          op[i] = *reinterpret_cast<const float4*>(rec + r * kDim + chunk);
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) to = fmaxf(to, mp[i]);
      const float old = m == -INFINITY ? 0.f : exp2f(m - to);
      m = to;
      l = __fmul_rn(l, old);
      o.x = __fmul_rn(o.x, old); o.y = __fmul_rn(o.y, old);
      o.z = __fmul_rn(o.z, old); o.w = __fmul_rn(o.w, old);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (mp[i] == -INFINITY) continue;  // no run, or one of which the row saw nothing
        const float w = exp2f(mp[i] - m);
        o.x = __fmaf_rn(w, op[i].x, o.x); o.y = __fmaf_rn(w, op[i].y, o.y);
        o.z = __fmaf_rn(w, op[i].z, o.z); o.w = __fmaf_rn(w, op[i].w, o.w);
        l = __fmaf_rn(w, lp[i], l);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const uint32_t token = row / a.group, h = head * a.group + row % a.group;
    T* out = static_cast<T*>(a.out.data) + (uint64_t)(s.q0 + token) * a.out.row_stride +
             h * a.out.head_stride + chunk;
    store4(out, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
  }
}

// The trees' second launch, which may begin while the first ends.
template <class T, int kDim, int kRows, int kKeys, int kLeast>
uint32_t launch_combine(const AttnArgs& a, uint32_t grid, cudaStream_t s) {
  constexpr int kStep = 256 / (kDim / 4);
  const dim3 join(grid, std::min(4, (kRows + kStep - 1) / kStep));
  PB_CUDA(launch_pdl(combine_kernel<T, kDim, kRows, kKeys, kLeast>, join, 256, a.seqs * 4, s, a, grid));
  return PB_OK;
}

}  // namespace paged
}  // namespace pb
