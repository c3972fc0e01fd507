// Pages of a paged key/value cache: the host's counted book of them, and the
// device copies behind forks and compaction and the kept path of a draft tree.
#include "pb_common.cuh"
#include "pb_paged.cuh"

#include <algorithm>
#include <new>
#include <vector>

namespace pb {
namespace {

using paged::refuse;

// A page's heads, slots and elements are contiguous per layer, for keys and for
// values, so a copy of n pages is n * layers * 2 contiguous pieces.  A warp moves
// 32 * U words of 16 bytes of one piece at a time, all U loads before the stores;
// bound by memory, one read and one write of each byte.
template <int U>
__global__ void __launch_bounds__(256) copy_pages_kernel(uint8_t* k, uint8_t* v,
                                                         uint64_t layer_bytes, uint32_t pages,
                                                         uint32_t page_words, uint32_t layers,
                                                         const uint32_t* pairs, uint64_t units) {
  const uint32_t parts = page_words / (32 * U);
  const uint64_t warps = (uint64_t)gridDim.x * 8;
  for (uint64_t u = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += warps) {
    const uint32_t part = (uint32_t)(u % parts);
    uint64_t rest = u / parts;
    const uint32_t side = (uint32_t)(rest & 1);
    rest >>= 1;
    const uint32_t layer = (uint32_t)(rest % layers);
    const uint64_t pair = rest / layers;
    const uint32_t from = pairs[2 * pair], to = pairs[2 * pair + 1];
    if (from >= pages || to >= pages) continue;
    uint4* base = reinterpret_cast<uint4*>((side ? v : k) + layer * layer_bytes) + part * (32 * U) +
                  (threadIdx.x & 31);
    const uint4* src = base + (uint64_t)from * page_words;
    uint4* dst = base + (uint64_t)to * page_words;
    uint4 w[U];
#pragma unroll
    for (int i = 0; i < U; ++i) w[i] = src[32 * i];
#pragma unroll
    for (int i = 0; i < U; ++i) dst[32 * i] = w[i];
  }
}

struct KeepArgs {
  uint8_t *k, *v;
  uint64_t layer_bytes;
  uint32_t layers, pages, page_size, kv_heads, row_words;
  const uint32_t *tables, *contexts, *counts, *nodes;
  uint32_t table_width, nodes_width;
  uint32_t columns;  // layers * 2 * kv_heads * row_words
};

// One CTA per sequence and 128 of its columns (layer, keys or values, head, 16-byte
// word of a row).  Its threads first work out the moves together, each a source and a
// target row, then each makes all moves of its column by itself, so that the moves
// need no order between threads.  Within a column the kept node indices n_i ascend
// and n_i >= i, so target i never equals the source of a later move (n_k > n_i >= i):
// sources are read kBatch at a time before their targets are written.  Bound by the
// latency of its three dependent loads (node, page, row) where it is small, else by
// memory.
constexpr int kBatch = 8, kMoves = 128;
__global__ void __launch_bounds__(128) keep_kernel(const __grid_constant__ KeepArgs a) {
  __shared__ uint32_t sources[kMoves], targets[kMoves];  // rows of head 0 in units of page slots; PB_NONE: no move
  __shared__ int64_t warp_top[4];
  __shared__ uint32_t warp_moves[4];
  const uint32_t seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t column = blockIdx.x * 128 + tid;
  const uint32_t* table = a.tables + (uint64_t)seq * a.table_width;
  const uint32_t* nodes = a.nodes + (uint64_t)seq * a.nodes_width;
  const uint64_t reach = (uint64_t)a.table_width * a.page_size;
  const uint32_t word = column % a.row_words;
  uint32_t rest = column / a.row_words;
  const uint32_t head = rest % a.kv_heads;
  rest /= a.kv_heads;
  uint4* base = reinterpret_cast<uint4*>((rest & 1 ? a.v : a.k) + (rest >> 1) * a.layer_bytes) +
                (uint64_t)head * a.page_size * a.row_words + word;
  int64_t top = -1;  // the largest node so far
  uint32_t count = 0xffffffffu;
  for (uint32_t i0 = 0; i0 < a.nodes_width && i0 < count; i0 += kMoves) {
    const uint32_t i = i0 + tid;
    const int64_t n = i < a.nodes_width ? (int64_t)nodes[i] : -1;
    const uint64_t context = a.contexts[seq];
    count = a.counts[seq];
    if (count == PB_NONE) count = 0;
    // the largest node before this one, over the warp and then the block
    int64_t before = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before = max(before, o);
    }
    __syncthreads();  // the moves before have been read
    if (lane == 31) warp_top[warp] = before;
    int64_t up_to = __shfl_up_sync(0xffffffffu, before, 1);
    if (lane == 0) up_to = -1;
    __syncthreads();
    up_to = max(up_to, top);
    for (uint32_t w = 0; w < 4; ++w) {
      if (w < warp) up_to = max(up_to, warp_top[w]);
      top = max(top, warp_top[w]);
    }
    bool move = i < count && i < a.nodes_width && n > (int64_t)i && n > up_to;  // n = i stays where it is
    uint32_t from = PB_NONE, to = PB_NONE;
    if (move && context + (uint64_t)n < reach) {
      const uint64_t src = context + (uint64_t)n, dst = context + i;
      const uint32_t p0 = table[src / a.page_size], p1 = table[dst / a.page_size];
      if (p0 < a.pages && p1 < a.pages) {
        from = p0 * a.page_size + (uint32_t)(src % a.page_size);
        to = p1 * a.page_size + (uint32_t)(dst % a.page_size);
      }
    }
    // only the moves, in their order
    move = from != PB_NONE;
    const uint32_t vote = __ballot_sync(0xffffffffu, move);
    if (lane == 0) warp_moves[warp] = __popc(vote);
    __syncthreads();
    uint32_t at = __popc(vote & ((1u << lane) - 1u)), moves = 0;
    for (uint32_t w = 0; w < 4; ++w) {
      if (w < warp) at += warp_moves[w];
      moves += warp_moves[w];
    }
    if (move) {
      sources[at] = from;
      targets[at] = to;
    }
    __syncthreads();
    if (column < a.columns) {
      auto row = [&](uint32_t spot) -> uint4* {
        const uint32_t page = spot / a.page_size;
        return base + ((uint64_t)page * a.kv_heads * a.page_size + spot % a.page_size) * a.row_words;
      };
      for (uint32_t m0 = 0; m0 < moves; m0 += kBatch) {
        uint4 w[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (m0 + j < moves) w[j] = *row(sources[m0 + j]);
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (m0 + j < moves) *row(targets[m0 + j]) = w[j];
      }
    }
  }
}

}  // namespace
}  // namespace pb

// ------------------------------------------------------------- the host's book

struct pb_pool {
  struct Sequence {
    bool open = false;
    uint32_t length = 0;
    std::vector<uint32_t> pages;
  };
  uint32_t page_size = 0, free_count = 0, max_seqs = 0;
  std::vector<uint32_t> holders;  // sequences that hold each page
  std::vector<uint32_t> free_ids;  // the first free_count entries; sized for all pages
  std::vector<Sequence> seqs;  // as many as were ever open at once, max_seqs at most

  bool is_open(uint32_t s) const { return s < seqs.size() && seqs[s].open; }
  void drop(uint32_t page) {
    if (--holders[page] == 0) free_ids[free_count++] = page;
  }
  uint32_t take() {
    const uint32_t page = free_ids[--free_count];
    holders[page] = 1;
    return page;
  }
};

namespace {
uint32_t not_open(const char* who) { return pb::paged::refuse(PB_STATE, who, "the sequence is not open"); }
uint32_t no_memory(const char* who) { return pb::paged::refuse(PB_CAPACITY, who, "out of host memory"); }
}  // namespace

extern "C" {

uint32_t pb_cache_copy_pages_device(const pb_cache* cache, uint32_t n, const uint32_t* pairs,
                                    void* stream) {
  const char* who = "pb_cache_copy_pages_device";
  uint32_t st;
  if ((st = pb::paged::check_cache(cache, who))) return st;
  if (n == 0) return PB_OK;
  if (!pairs) return pb::paged::refuse(PB_CAPACITY, who, "pairs is NULL");
  const uint32_t bytes = pb::paged::type_bytes(cache->type);
  const uint32_t page_words = cache->kv_heads * cache->page_size * cache->head_dim * bytes / 16;
  const uint32_t unroll = page_words % 128 == 0 ? 4 : 1;
  const uint64_t units = (uint64_t)n * cache->layers * 2 * (page_words / (32 * unroll));
  const uint32_t grid = (uint32_t)std::min<uint64_t>((units + 7) / 8, 0x7fffffffu);
  auto* k = static_cast<uint8_t*>(cache->k);
  auto* v = static_cast<uint8_t*>(cache->v);
  auto kernel = unroll == 4 ? pb::copy_pages_kernel<4> : pb::copy_pages_kernel<1>;
  kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(k, v, cache->layer_stride * bytes, cache->pages,
                                                 page_words, cache->layers, pairs, units);
  PB_CUDA(cudaGetLastError());
  return PB_OK;
}

uint32_t pb_cache_keep_device(const pb_cache* cache, uint32_t seqs, const uint32_t* tables,
                              uint32_t table_width, const uint32_t* contexts,
                              const uint32_t* counts, const uint32_t* nodes, uint32_t nodes_width,
                              void* stream) {
  const char* who = "pb_cache_keep_device";
  uint32_t st;
  if ((st = pb::paged::check_cache(cache, who))) return st;
  if (seqs == 0 || nodes_width == 0) return PB_OK;
  if (!tables || !table_width || !contexts || !counts || !nodes)
    return pb::paged::refuse(PB_CAPACITY, who, "an empty table or a NULL argument");
  const uint32_t bytes = pb::paged::type_bytes(cache->type);
  pb::KeepArgs a{};
  a.k = static_cast<uint8_t*>(cache->k);
  a.v = static_cast<uint8_t*>(cache->v);
  a.layer_bytes = cache->layer_stride * bytes;
  a.layers = cache->layers; a.pages = cache->pages; a.page_size = cache->page_size;
  a.kv_heads = cache->kv_heads; a.row_words = cache->head_dim * bytes / 16;
  a.tables = tables; a.contexts = contexts; a.counts = counts; a.nodes = nodes;
  a.table_width = table_width; a.nodes_width = nodes_width;
  const uint64_t columns = (uint64_t)a.layers * 2 * a.kv_heads * a.row_words;
  if (columns >= 1u << 31) return pb::paged::refuse(PB_CAPACITY, who, "too many layers");
  a.columns = (uint32_t)columns;
  // grid.y holds 65535 sequences: further ones in further launches
  for (uint32_t s0 = 0; s0 < seqs; s0 += 65535) {
    const uint32_t n = std::min<uint32_t>(65535, seqs - s0);
    pb::keep_kernel<<<dim3((a.columns + 127) / 128, n), 128, 0, (cudaStream_t)stream>>>(a);
    a.tables += (uint64_t)n * table_width;
    a.contexts += n;
    a.counts += n;
    a.nodes += (uint64_t)n * nodes_width;
  }
  PB_CUDA(cudaGetLastError());
  return PB_OK;
}

uint32_t pb_pool_create(uint32_t pages, uint32_t page_size, uint32_t max_seqs, pb_pool** out) {
  const char* who = "pb_pool_create";
  if (!out) return pb::paged::refuse(PB_CAPACITY, who, "out is NULL");
  *out = nullptr;
  if (!pages || pages >= 1u << 31 || !page_size || !max_seqs ||
      (uint64_t)pages * page_size >= 1ull << 31)
    return pb::paged::refuse(PB_CAPACITY, who, "pages, page_size and max_seqs must be positive, pages * page_size below 2^31");
  pb_pool* p = new (std::nothrow) pb_pool();
  if (!p) return no_memory(who);
  try {
    p->page_size = page_size;
    p->max_seqs = max_seqs;
    p->holders.assign(pages, 0);
    p->free_ids.resize(pages);
  } catch (...) {
    delete p;
    return no_memory(who);
  }
  // the lowest ids are given out first
  for (uint32_t i = 0; i < pages; ++i) p->free_ids[i] = pages - 1 - i;
  p->free_count = pages;
  *out = p;
  return PB_OK;
}

void pb_pool_destroy(pb_pool* pool) { delete pool; }

uint32_t pb_pool_open(pb_pool* p, uint32_t* seq) {
  const char* who = "pb_pool_open";
  if (!p || !seq) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  for (uint32_t s = 0; s < p->seqs.size(); ++s)
    if (!p->seqs[s].open) {
      p->seqs[s].open = true;
      p->seqs[s].length = 0;
      p->seqs[s].pages.clear();
      *seq = s;
      return PB_OK;
    }
  if (p->seqs.size() >= p->max_seqs) return pb::paged::refuse(PB_CAPACITY, who, "every sequence is open");
  try {
    p->seqs.emplace_back();
  } catch (...) {
    return no_memory(who);
  }
  p->seqs.back().open = true;
  *seq = (uint32_t)p->seqs.size() - 1;
  return PB_OK;
}

uint32_t pb_pool_fork(pb_pool* p, uint32_t seq, uint32_t* child) {
  const char* who = "pb_pool_fork";
  if (!p || !child) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  if (!p->is_open(seq)) return not_open(who);
  uint32_t s = 0;
  uint32_t st = pb_pool_open(p, &s);
  if (st) return st;
  try {
    p->seqs[s].pages = p->seqs[seq].pages;
  } catch (...) {
    p->seqs[s].open = false;
    return no_memory(who);
  }
  p->seqs[s].length = p->seqs[seq].length;
  for (uint32_t page : p->seqs[s].pages) ++p->holders[page];
  *child = s;
  return PB_OK;
}

uint32_t pb_pool_extend(pb_pool* p, uint32_t seq, uint32_t tokens, uint32_t* pair,
                        uint32_t* needed) {
  const char* who = "pb_pool_extend";
  if (!p || !pair) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  if (!p->is_open(seq)) return not_open(who);
  pb_pool::Sequence& q = p->seqs[seq];
  const uint64_t length = (uint64_t)q.length + tokens;
  const uint64_t want = (length + p->page_size - 1) / p->page_size;
  const bool split = tokens && q.length % p->page_size && p->holders[q.pages.back()] > 1;
  const uint64_t fresh = want - q.pages.size() + split;
  if (fresh > p->free_count) {
    if (needed) *needed = (uint32_t)std::min<uint64_t>(fresh, PB_NONE);
    return pb::paged::refuse(PB_CAPACITY, who, "too few free pages");
  }
  try {
    q.pages.reserve((size_t)want);
  } catch (...) {
    return no_memory(who);
  }
  pair[0] = pair[1] = PB_NONE;
  if (split) {
    pair[0] = q.pages.back();
    pair[1] = p->take();
    p->drop(pair[0]);
    q.pages.back() = pair[1];
  }
  while (q.pages.size() < want) q.pages.push_back(p->take());
  q.length = (uint32_t)length;
  if (needed) *needed = (uint32_t)fresh;
  return PB_OK;
}

uint32_t pb_pool_truncate(pb_pool* p, uint32_t seq, uint32_t length) {
  const char* who = "pb_pool_truncate";
  if (!p) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  if (!p->is_open(seq)) return not_open(who);
  pb_pool::Sequence& q = p->seqs[seq];
  if (length > q.length) return pb::paged::refuse(PB_CAPACITY, who, "the sequence is shorter than that");
  const size_t want = ((size_t)length + p->page_size - 1) / p->page_size;
  while (q.pages.size() > want) {
    p->drop(q.pages.back());
    q.pages.pop_back();
  }
  q.length = length;
  return PB_OK;
}

uint32_t pb_pool_free(pb_pool* p, uint32_t seq) {
  const char* who = "pb_pool_free";
  if (!p) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  if (!p->is_open(seq)) return not_open(who);
  uint32_t st = pb_pool_truncate(p, seq, 0);
  if (st) return st;
  p->seqs[seq].open = false;
  return PB_OK;
}

uint32_t pb_pool_compact(pb_pool* p, uint32_t* pairs, uint32_t capacity, uint32_t* n, uint32_t* used,
                         uint32_t* needed) {
  const char* who = "pb_pool_compact";
  if (!p || !n || !used) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  const uint32_t pages = (uint32_t)p->holders.size();
  const uint32_t live = pages - p->free_count;
  uint32_t moves = 0;  // the pages in use past the first `live`
  for (uint32_t i = live; i < pages; ++i) moves += p->holders[i] != 0;
  if (needed) *needed = moves;
  if (moves > capacity || (moves && !pairs))
    return pb::paged::refuse(PB_CAPACITY, who, "the array of pairs is too short");
  std::vector<uint32_t> now;
  try {
    now.resize(pages);
  } catch (...) {
    return no_memory(who);
  }
  uint32_t hole = 0, at = 0;
  for (uint32_t i = 0; i < pages; ++i) now[i] = i;
  for (uint32_t i = live; i < pages; ++i) {
    if (!p->holders[i]) continue;
    while (p->holders[hole]) ++hole;  // a hole below `live` exists for each of them
    pairs[2 * at] = i;
    pairs[2 * at + 1] = hole;
    ++at;
    p->holders[hole] = p->holders[i];
    p->holders[i] = 0;
    now[i] = hole;
  }
  for (auto& q : p->seqs)
    for (uint32_t& page : q.pages) page = now[page];
  for (uint32_t i = 0; i < p->free_count; ++i) p->free_ids[i] = pages - 1 - i;
  *n = moves;
  *used = live;
  return PB_OK;
}

uint32_t pb_pool_table(const pb_pool* p, uint32_t seq, uint32_t* table, uint32_t width,
                       uint32_t* length, uint32_t* needed) {
  const char* who = "pb_pool_table";
  if (!p || (!table && width)) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  if (!p->is_open(seq)) return not_open(who);
  const pb_pool::Sequence& q = p->seqs[seq];
  if (needed) *needed = (uint32_t)q.pages.size();
  if (q.pages.size() > width) return pb::paged::refuse(PB_CAPACITY, who, "the table is too short");
  std::copy(q.pages.begin(), q.pages.end(), table);
  std::fill(table + q.pages.size(), table + width, PB_NONE);
  if (length) *length = q.length;
  return PB_OK;
}

uint32_t pb_pool_free_pages(const pb_pool* p) { return p ? p->free_count : 0; }

}  // extern "C"
