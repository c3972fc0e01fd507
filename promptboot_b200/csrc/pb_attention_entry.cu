// C entries of the paged serving attention: argument checks and the choice of
// kernel.
#include "pb_attention_launch.h"
#include "pb_common.cuh"
#include "pb_told.h"

#include <cmath>

namespace pb {
namespace paged {

uint32_t tree_ctas(uint32_t per_sm) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return (uint32_t)sms * per_sm;
}

namespace {

uint32_t check_heads(const char* who, uint32_t type, uint32_t head_dim, uint32_t q_heads,
                     uint32_t kv_heads, uint32_t seqs, uint32_t rows) {
  if (!type_bytes(type)) return refuse(PB_CAPACITY, who, "unknown element type");
  if (head_dim != 64 && head_dim != 128) return refuse(PB_CAPACITY, who, "head_dim must be 64 or 128");
  if (!q_heads || q_heads > 1024 || !kv_heads || q_heads % kv_heads)
    return refuse(PB_CAPACITY, who, "q_heads must be a multiple of kv_heads, up to 1024");
  if (!seqs || seqs > PB_MAX_SEQS) return refuse(PB_CAPACITY, who, "1 to 2048 sequences");
  if ((uint64_t)rows * q_heads >= 1ull << 30)
    return refuse(PB_CAPACITY, who, "rows * q_heads must stay below 2^30");
  return PB_OK;
}

constexpr float kLog2E = 1.4426950408889634f;

uint32_t check_scale(const char* who, float scale) {
  if (!(scale > 0.f) || !std::isfinite(scale * kLog2E))
    return refuse(PB_CAPACITY, who, "scale must be positive and scale * log2(e) finite");
  return PB_OK;
}

// Row groups of 16 that hold a sequence's rows of one key head on average: 1, or 2 at
// heads of 64 (at heads of 128 their sums would not fit the registers); 0 where they
// are more.
uint32_t few_tiles(uint32_t head_dim, uint64_t rows, uint32_t seqs) {
  if (rows <= 16ull * seqs) return 1;
  return head_dim == 64 && rows <= 32ull * seqs ? 2 : 0;
}

// Row tile of the binary32 kernel for few rows that holds a sequence's rows of one key
// head on average, 0 where they are more than 16.
uint32_t few32_rows(uint64_t rows, uint32_t seqs) {
  if (rows <= 8ull * seqs) return 8;
  return rows <= 16ull * seqs ? 16 : 0;
}

}  // namespace
}  // namespace paged
}  // namespace pb

using pb::paged::refuse;

extern "C" {

uint32_t pb_prompt_attention_device(uint32_t type, uint32_t head_dim, uint32_t q_heads,
                                    uint32_t kv_heads, uint32_t seqs, uint32_t q_rows,
                                    uint32_t kv_rows, const pb_rows* q, const pb_rows* k,
                                    const pb_rows* v, const pb_rows* out, const uint32_t* q_offsets,
                                    const uint32_t* kv_offsets, float scale, void* stream) {
  const char* who = "pb_prompt_attention_device";
  uint32_t st;
  if ((st = pb::paged::check_heads(who, type, head_dim, q_heads, kv_heads, seqs, q_rows))) return st;
  if ((st = pb::paged::check_scale(who, scale))) return st;
  const uint32_t bytes = pb::paged::type_bytes(type);
  if (!q_rows) return PB_OK;
  if (kv_rows >= 1u << 30) return refuse(PB_CAPACITY, who, "kv_rows must stay below 2^30");
  if (!kv_offsets && kv_rows != q_rows)
    return refuse(PB_CAPACITY, who, "other key rows than q rows need kv_offsets");
  if (!q_offsets) return refuse(PB_CAPACITY, who, "q_offsets is NULL");
  if ((st = pb::paged::check_rows(q, bytes, who, "q"))) return st;
  if (!kv_rows) k = v = q;  // not read: without key rows they may be NULL
  if ((st = pb::paged::check_rows(k, bytes, who, "k"))) return st;
  if ((st = pb::paged::check_rows(v, bytes, who, "v"))) return st;
  if ((st = pb::paged::check_output(out, bytes, q_rows, q_heads, who, "out"))) return st;
  if (kv_rows > 1 && (!k->row_stride || !v->row_stride))
    return refuse(PB_CAPACITY, who, "k and v need a row stride");
  pb::paged::AttnArgs a{};
  a.q = *q; a.k = *k; a.v = *v; a.out = *out;
  a.q_offsets = q_offsets;
  a.kv_offsets = kv_offsets ? kv_offsets : q_offsets;
  a.seqs = seqs; a.q_rows = q_rows; a.kv_rows = kv_rows;
  a.kv_heads = kv_heads; a.group = q_heads / kv_heads;
  a.scale_log2 = scale * pb::paged::kLog2E;
  if (bytes == 2) return pb::paged::tc_prompt(a, type, head_dim, (cudaStream_t)stream);
  return pb::paged::simt_prompt(a, head_dim, (cudaStream_t)stream);
}

uint64_t pb_tree_attention_workspace(uint32_t type, uint32_t head_dim, uint32_t q_heads,
                                     uint32_t kv_heads, uint32_t seqs, uint32_t rows) {
  if (pb::paged::check_heads("pb_tree_attention_workspace", type, head_dim, q_heads, kv_heads, seqs, rows))
    return 0;
  const uint64_t all = (uint64_t)rows * (q_heads / kv_heads);
  if (type == PB_TYPE_F32) {
    const uint32_t tile = pb::paged::few32_rows(all, seqs);
    return (tile ? pb::paged::few32_tree_words(head_dim, tile) : pb::paged::simt_tree_words(head_dim)) * 4;
  }
  const uint32_t tiles = pb::paged::few_tiles(head_dim, all, seqs);
  return (tiles ? pb::paged::few_tree_words(head_dim, tiles) : pb::paged::tc_tree_words(head_dim)) * 4;
}

uint32_t pb_tree_attention_device(const pb_cache* cache, uint32_t layer, uint32_t q_heads,
                                  uint32_t seqs, uint32_t rows, const pb_rows* q,
                                  const pb_rows* out, const uint32_t* tables, uint32_t table_width,
                                  const uint32_t* contexts, const uint32_t* offsets,
                                  const uint64_t* visible, float scale, void* workspace,
                                  uint64_t workspace_bytes, void* stream) {
  const char* who = "pb_tree_attention_device";
  uint32_t st;
  if ((st = pb::paged::check_cache(cache, who))) return st;
  if (layer >= cache->layers) return refuse(PB_CAPACITY, who, "no such layer");
  if ((st = pb::paged::check_heads(who, cache->type, cache->head_dim, q_heads, cache->kv_heads, seqs, rows)))
    return st;
  if ((st = pb::paged::check_scale(who, scale))) return st;
  if (!rows) return PB_OK;
  const uint32_t bytes = pb::paged::type_bytes(cache->type);
  if ((st = pb::paged::check_rows(q, bytes, who, "q"))) return st;
  if ((st = pb::paged::check_output(out, bytes, rows, q_heads, who, "out"))) return st;
  if (!tables || !table_width || !contexts || !offsets || !visible)
    return refuse(PB_CAPACITY, who, "an empty table or a NULL argument");
  // Key tiles are counted in 32 bits: of `least` keys or more, for row tiles of `least` or more.
  const uint64_t group = q_heads / cache->kv_heads, reach = (uint64_t)table_width * cache->page_size;
  const uint32_t least = bytes == 4 ? 8 : 16;
  const uint64_t segments = (rows * group / least + seqs) * cache->kv_heads;
  if (reach >= 1ull << 30 || segments * (reach / least + 1) >= 1ull << 31)
    return refuse(PB_CAPACITY, who, "the tables reach too far for so many sequences and rows");
  const uint64_t need = pb_tree_attention_workspace(cache->type, cache->head_dim, q_heads,
                                                    cache->kv_heads, seqs, rows);
  if (!workspace || workspace_bytes < need)
    return refuse(PB_CAPACITY, who, "the workspace is smaller than pb_tree_attention_workspace says");
  if (!pb::paged::aligned16(workspace)) return refuse(PB_ALIGNMENT, who, "the workspace needs 16-byte alignment");
  pb::paged::AttnArgs a{};
  a.q = *q; a.out = *out;
  a.cache = pb::paged::layer_view(cache, layer);
  a.q_offsets = offsets; a.tables = tables; a.contexts = contexts;
  a.visible = reinterpret_cast<const unsigned long long*>(visible);
  a.seqs = seqs; a.q_rows = rows;
  a.kv_heads = cache->kv_heads; a.group = (uint32_t)group; a.table_width = table_width;
  a.scale_log2 = scale * pb::paged::kLog2E;
  a.partial = static_cast<float*>(workspace);
  if (bytes == 2) {
    const uint32_t tiles = pb::paged::few_tiles(cache->head_dim, rows * group, seqs);
    return tiles ? pb::paged::few_tree(a, cache->type, cache->head_dim, tiles, (cudaStream_t)stream)
                 : pb::paged::tc_tree(a, cache->type, cache->head_dim, (cudaStream_t)stream);
  }
  if (const uint32_t tile = pb::paged::few32_rows(rows * group, seqs))
    return pb::paged::few32_tree(a, cache->head_dim, tile, (cudaStream_t)stream);
  return pb::paged::simt_tree(a, cache->head_dim, (cudaStream_t)stream);
}

uint32_t pb_attention_status(void* stream) {
  static thread_local pb::Told told;
  const cudaStream_t s = (cudaStream_t)stream;
  uint32_t st, count = 0;
  if ((st = pb::paged::tc_timeouts(s, &count))) return st;
  if ((st = pb::paged::few_timeouts(s, &count))) return st;
  if ((st = pb::paged::few32_timeouts(s, &count))) return st;
  int device = 0;
  PB_CUDA(cudaGetDevice(&device));
  if (!told.news(device, count)) return PB_OK;
  pb::set_last_error("an attention pipeline timed out waiting for a copy or a product");
  return PB_DEVICE;
}

}  // extern "C"
