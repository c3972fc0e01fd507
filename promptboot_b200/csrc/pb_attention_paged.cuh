// Work division of the paged serving attention, shared by its kernels.
//
// Rows are packed: the rows of one (sequence, key head) are its tokens or nodes
// times the query heads that share the key head, row r = token * group + head, so
// that grouped heads and short sequences fill a row tile.  A row tile of one
// (sequence, key head) is a segment; its keys are walked in tiles.
//
// Prompts: one CTA per segment, the row tiles of a sequence from its end (the
// longest) to its start.  Trees: all key tiles of all segments form one list,
// which is shared out evenly in consecutive runs, one to a CTA or a warp, whatever the
// sequences' lengths are; a segment that crosses runs leaves one partial (weighted sum,
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
  float* partial;    // trees: two records a run
  struct Join* joins;  // and what is to be joined where a run ends
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

// The largest; not a number where one is not.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

__host__ __device__ __forceinline__ uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

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

// The trees' list of `total` key tiles in `most` runs, at least kLeast tiles each: run
// c is [start(c), start(c + 1)), and tile x is in run holder(x).  A run is a CTA's, or
// a warp's in pb_attention_few.cu.
template <int kLeast>
struct Share {
  uint32_t total, runs;
  __device__ __forceinline__ Share(uint32_t total_, uint32_t most)
      : total(total_), runs(min(most, max(1u, total_ / kLeast))) {}
  __device__ __forceinline__ uint32_t start(uint32_t c) const {
    return (uint32_t)((uint64_t)c * total / runs);
  }
  __device__ __forceinline__ uint32_t holder(uint32_t x) const {
    return (uint32_t)((((uint64_t)x + 1) * runs - 1) / total);
  }
};

// A run of key tiles [tile0, tile1) of one segment.
struct Piece {
  uint32_t seq, head, row_tile;
  uint32_t tile0, tile1;
  int partial;  // workspace record, -1: the whole segment, straight to out
};

// The partial of run c for a segment that began before it, or that begins in it.
__device__ __forceinline__ int partial_of(uint32_t run, bool begins) { return (int)(2 * run + begins); }

// Takes the next piece of run `run`'s items [next, end).
template <bool kTree, int kRows, int kKeys>
__device__ __forceinline__ void take_piece(const AttnArgs& a, const uint32_t* prefix, uint32_t run, uint32_t& next,
                                           uint32_t end, Piece& p, Sequence& s, uint32_t& rows) {
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
    if (p.tile0 > 0 || p.tile1 < tiles) p.partial = partial_of(run, p.tile0 == 0);
    next += p.tile1 - p.tile0;
  } else {
    p.head = x % a.kv_heads;
    p.row_tile = row_tiles - 1 - x / a.kv_heads;
    const uint32_t last = min(rows, (p.row_tile + 1) * kRows) - 1;
    p.tile0 = 0;
    p.tile1 = ceil_div(row_view<false>(a, s, last / a.group).all, kKeys);
    ++next;
  }
  // Offsets that do not ascend can make the work overflow its counters: what is then no
  // segment has no rows and no tiles.
  if (p.row_tile >= row_tiles || p.head >= a.kv_heads) rows = 0;
  if (rows == 0 || s.len == 0) p.tile1 = p.tile0 = 0;  // nothing to see
}

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

// The segment that begins in a run and goes on in the next: its last run, the rows of
// its sequence from q0 on, its head and row tile.  last PB_NONE: there is none.
struct alignas(16) Join {
  uint32_t last, q0, rows, head, row_tile;
};

// Notes the segment that crosses the end of run `run` (one thread of it, every run of
// the launch).
template <int kRows, int kKeys, int kLeast>
__device__ __forceinline__ void note_join(const AttnArgs& a, const uint32_t* prefix, const Share<kLeast>& share,
                                          uint32_t run) {
  Join j{PB_NONE, 0, 0, 0, 0};
  if (share.total > 0 && run + 1 < share.runs) {
    const uint32_t edge = share.start(run + 1);
    uint32_t x = edge;
    const Sequence s = load_sequence<true>(a, find_sequence(prefix, a.seqs, x));
    const uint32_t tiles = max(1u, ceil_div(s.len, kKeys)), begin = edge - x % tiles;
    const uint32_t rows = s.t * a.group, row_tiles = max(1u, ceil_div(rows, kRows));
    const uint32_t head = x / tiles / row_tiles;
    // else it begins at the edge, or in an earlier run (or is none: see take_piece)
    if (begin != edge && begin >= share.start(run) && head < a.kv_heads)
      j = {min(share.holder(begin + tiles - 1), share.runs - 1), s.q0, rows, head, x / tiles % row_tiles};
  }
  a.joins[run] = j;
}

// Joins the partials of the segments that crossed runs: weights 2^(m_i - m), in the
// order of the runs, so the result does not depend on timing.  A segment is joined by
// the CTAs of the run in which it begins.  A thread has four elements of a row and loads
// eight partials at a time: latency is what there is to save here.
constexpr int kCombine = 128;  // threads
template <class T, int kDim, int kRows>
__global__ void __launch_bounds__(kCombine) combine_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();  // the notes and the partials
  const uint32_t c = blockIdx.x;
  const Join j = a.joins[c];
  if (j.last == PB_NONE) return;
  constexpr int kPerRow = kDim / 4, kStep = kCombine / kPerRow, kBatch = 8;
  const int chunk = (threadIdx.x % kPerRow) * 4;
  for (uint32_t r = blockIdx.y * kStep + threadIdx.x / kPerRow; r < kRows; r += gridDim.y * kStep) {
    const uint32_t row = j.row_tile * kRows + r;
    if (row >= j.rows) return;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t p0 = c; p0 <= j.last; p0 += kBatch) {
      float mp[kBatch], lp[kBatch];
      float4 op[kBatch];
      float to = m;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        mp[i] = -INFINITY;
        if (p0 + i <= j.last) {
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
        // no run, or one of which the row saw nothing (a score that is not a number makes
        // the run's maximum one that is not)
        if (mp[i] == -INFINITY) continue;
        const float w = exp2f(mp[i] - m);
        o.x = __fmaf_rn(w, op[i].x, o.x); o.y = __fmaf_rn(w, op[i].y, o.y);
        o.z = __fmaf_rn(w, op[i].z, o.z); o.w = __fmaf_rn(w, op[i].w, o.w);
        l = __fmaf_rn(w, lp[i], l);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const uint32_t token = row / a.group, h = j.head * a.group + row % a.group;
    T* out = static_cast<T*>(a.out.data) + (uint64_t)(j.q0 + token) * a.out.row_stride +
             h * a.out.head_stride + chunk;
    store4(out, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
  }
}

// The trees' second launch, which may begin while the first ends.
template <class T, int kDim, int kRows>
uint32_t launch_combine(const AttnArgs& a, uint32_t runs, cudaStream_t s) {
  constexpr uint32_t kStep = kCombine / (kDim / 4);
  // CTAs for the rows that a sequence has on average; those of longer ones take turns.
  const uint32_t mean = (uint32_t)(((uint64_t)a.q_rows * a.group + a.seqs - 1) / a.seqs);
  const dim3 join(runs, std::max(1u, ceil_div(std::min<uint32_t>(kRows, mean), kStep)));
  PB_CUDA(launch_pdl(combine_kernel<T, kDim, kRows>, join, kCombine, 0, s, a));
  return PB_OK;
}

// Words of a tree's workspace: two partials and a note per run.
inline uint64_t tree_words(uint64_t runs, uint64_t rows, uint64_t head_dim) {
  return runs * (2 * rows * (head_dim + 2) + sizeof(Join) / 4);
}
// Places them; the partials first.
inline void place_workspace(AttnArgs& a, uint64_t runs, uint64_t rows, uint64_t head_dim) {
  a.joins = reinterpret_cast<Join*>(a.partial + runs * 2 * rows * (head_dim + 2));
}

}  // namespace paged
}  // namespace pb
