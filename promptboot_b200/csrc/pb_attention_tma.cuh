// Shared by the paged serving attention kernels that take tiles by TMA: element
// formats, tensor maps of packed rows and of the paged cache, and small device parts.
#pragma once

#include "pb_attention_paged.cuh"
#include "pb_tcgen05.cuh"

#include <cuda.h>

namespace pb {
namespace paged {

template <class T>
struct Format;
template <>
struct Format<float> {
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  static constexpr float kSlack = 8.f;
};
template <>
struct Format<__half> {
  static constexpr uint32_t kCode = 0;  // instruction descriptor
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  static constexpr float kSlack = 4.f, kRaise = 10.f;  // weights stay below 2^14 of 65504
  static constexpr uint32_t kExponents = 0x7c007c00u;
  static constexpr int kDegree = 4;
};
template <>
struct Format<__nv_bfloat16> {
  static constexpr uint32_t kCode = 1;
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  static constexpr float kSlack = 8.f, kRaise = 0.f;
  static constexpr uint32_t kExponents = 0x7f807f80u;
  static constexpr int kDegree = 3;
};

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }


// One lane of the warp, for the instructions below: the whole warp runs them, with
// that lane's predicate, so that their operands stay in uniform registers (issued from
// a branch of one lane, four MMAs and their commit took 450 cycles).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is)
      :
      : "memory");
  return is;
}
__device__ __forceinline__ void expect_tx(uint32_t leader, uint64_t* bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %2, 0;\n\t"
      "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}"
      ::"r"(smem_u32(bar)), "r"(bytes), "r"(leader)
      : "memory");
}
// TMA tile loads: the innermost coordinate is 0 or 64 elements (128 bytes).
__device__ __forceinline__ void tma_3d(uint32_t leader, uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                       uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %6, 0;\n\t"
      "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t leader, uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                       int w, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %7, 0;\n\t"
      "@e cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n\t}"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)), "r"(leader)
      : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Part `part` of kParts of value row `key` of a tile in shared memory (column blocks of
// 128 bytes, kBlock apart, 128-byte swizzle): zeroed where it is past the keys; else
// what is not finite is zeroed.  Whether there was any.
template <class F, int kDim, int kBlock, int kParts>
__device__ __forceinline__ bool clean_value_row(uint8_t* tile, int key, int part, bool past) {
  constexpr int kWords = kDim / 8 / kParts;
  constexpr uint32_t kLowest = (F::kExponents & (0u - F::kExponents)) * 0x10001u;
  auto word = [&](int i) {
    const int c = part * kWords + i;
    return reinterpret_cast<uint4*>(tile + c / 8 * kBlock + key * 128 + ((c % 8) ^ (key & 7)) * 16);
  };
  uint32_t full = 0;  // all exponent bits set: one more carries into the sign's place
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if (past) {
      *word(i) = make_uint4(0, 0, 0, 0);
    } else {
      const uint4 x = *word(i);
      full |= ((x.x & F::kExponents) + kLowest) | ((x.y & F::kExponents) + kLowest) |
              ((x.z & F::kExponents) + kLowest) | ((x.w & F::kExponents) + kLowest);
    }
  }
  if (!(full & 0x80008000u)) return false;
#pragma unroll 1
  for (int i = 0; i < kWords; ++i) {
    uint4 x = *word(i);
    uint32_t* u = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t e = u[k] & F::kExponents;
      if ((e & 0xffffu) == (F::kExponents & 0xffffu)) u[k] &= 0xffff0000u;
      if ((e >> 16) == (F::kExponents >> 16)) u[k] &= 0xffffu;
    }
    *word(i) = x;
  }
  return true;
}

struct Maps {
  CUtensorMap k, v;
  uint32_t k_step, v_step;  // 0: one key head's rows serve all
};

// A warp's ring of key and value tiles over its run [begin, end) of a tree's tile list,
// which it fills itself: tile `load` goes to stage loaded % kStages, keys first, in
// column blocks of 128 bytes (kBlocks of them) of kKeys rows.  Its segment, (sequence,
// head) with tile 0 at seg0, is decoded where it changes; the page ids of a tile are
// fetched when the one before is sent for.
template <class T, int kRows, int kKeys, int kBlocks, int kStages>
struct TileRing {
  static constexpr int kBlock = kKeys * 128, kTile = kBlocks * kBlock;
  const AttnArgs& a;
  const Maps& maps;
  const uint32_t* prefix;
  uint64_t* full;  // one barrier per stage
  uint8_t* ring;
  uint32_t leader, size, load, end, seg0 = 0, seg1 = 0, seq = 0, head = 0, len = 0;
  int lane, loaded = 0, page = 0;

  __device__ __forceinline__ TileRing(const AttnArgs& a_, const Maps& maps_, const uint32_t* prefix_, uint64_t* full_,
                                      uint8_t* ring_, uint32_t begin, uint32_t end_)
      : a(a_), maps(maps_), prefix(prefix_), full(full_), ring(ring_), leader(elect_one()),
        size(min(a_.cache.page_size, (uint32_t)kKeys)), load(begin), end(end_), lane(threadIdx.x & 31) {
    look();
#pragma unroll
    for (int i = 0; i < kStages; ++i) send();
  }
  __device__ __forceinline__ uint8_t* keys(int tile) const { return ring + tile % kStages * 2 * kTile; }
  __device__ __forceinline__ void look() {  // decodes tile `load` and fetches its page ids
    if (load >= end) return;
    if (load >= seg1) {
      uint32_t x = load;
      seq = find_sequence(prefix, a.seqs, x);
      const Sequence q = load_sequence<true>(a, seq);
      const uint32_t tiles = max(1u, ceil_div(q.len, kKeys));
      len = q.len;
      head = x / tiles / max(1u, ceil_div(q.t * a.group, kRows));
      seg0 = load - x % tiles;
      seg1 = seg0 + tiles;
    }
    const uint32_t key = (load - seg0) * kKeys + lane * size;
    if (lane * size < kKeys && key < len)
      page = (int)a.tables[(uint64_t)seq * a.table_width + key / a.cache.page_size];
  }
  __device__ __forceinline__ void send() {  // sends for tile `load`
    while (load < end && (load - seg0) * kKeys >= len) {  // no keys, no tile to wait for
      ++load;
      look();
    }
    if (load >= end) return;
    const uint32_t key = (load - seg0) * kKeys, slot = key % a.cache.page_size;
    uint64_t* bar = &full[loaded % kStages];
    const uint32_t count = min((uint32_t)kKeys / size, ceil_div(len - key, size));
    const uint32_t to = smem_u32(keys(loaded));
    expect_tx(leader, bar, 2 * count * size * kBlocks * 128);
    for (uint32_t b = 0; b < count; ++b) {
      const int at = __shfl_sync(0xffffffffu, page, b);
#pragma unroll
      for (int c = 0; c < kBlocks; ++c) {
        const int x = c * (int)(128 / sizeof(T));
        tma_4d(leader, to + c * kBlock + b * size * 128, &maps.k, x, (int)slot, (int)head, at, bar);
        tma_4d(leader, to + kTile + c * kBlock + b * size * 128, &maps.v, x, (int)slot, (int)head, at, bar);
      }
    }
    ++loaded;
    ++load;
    look();
  }
  // On the way out: what was sent for after `used` tiles lands before the CTA exits.
  __device__ __forceinline__ void drain(int used) {
    for (int i = max(used, loaded - kStages); i < loaded; ++i)
      wait_drain(&full[i % kStages], (i / kStages) & 1, 50000000ull);
  }
};

// CTAs in which a bounded wait gave up (one count per source file and device).  Never
// cleared, so that whoever asks takes nothing from others who have still to ask.
static __device__ unsigned int g_timeouts;
__device__ __forceinline__ void mark_timeout() { atomicAdd(&g_timeouts, 1u); }
// Adds it to *count, once `s` is done with what it has.
static inline uint32_t add_timeouts(cudaStream_t s, uint32_t* count) {
  unsigned int n = 0;
  PB_CUDA(cudaMemcpyFromSymbolAsync(&n, g_timeouts, 4, 0, cudaMemcpyDeviceToHost, s));
  PB_CUDA(cudaStreamSynchronize(s));
  *count += n;
  return PB_OK;
}

// --------------------------------------------------------------- tensor maps (host)

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                            const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                            CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline uint32_t encoder(Encode* out) {
  static std::atomic<Encode> known{nullptr};
  Encode found = known.load();
  if (!found) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult how;
    PB_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &how));
    if (how != cudaDriverEntryPointSuccess || !f) {
      set_last_error("the driver has no cuTensorMapEncodeTiled");
      return PB_DEVICE;
    }
    found = reinterpret_cast<Encode>(f);
    known.store(found);
  }
  *out = found;
  return PB_OK;
}

inline uint32_t encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, void* data, const cuuint64_t* dims,
                           const cuuint64_t* strides, const cuuint32_t* box) {
  Encode encode = nullptr;
  uint32_t st = encoder(&encode);
  if (st) return st;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult e = encode(map, type, rank, data, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (e == CUDA_SUCCESS) return PB_OK;
  char text[96];
  std::snprintf(text, sizeof text, "cuTensorMapEncodeTiled refused the keys or values (error %d)", (int)e);
  set_last_error(text);
  return PB_DEVICE;
}

// Keys and values of a cache layer: (element, slot, head, page), boxes of 128 bytes of
// one page's slots.
template <class T>
uint32_t cache_maps(const AttnArgs& a, uint32_t head_dim, uint32_t tile_keys, Maps* maps) {
  const cuuint64_t dim = head_dim, size = a.cache.page_size;
  const cuuint64_t dims[4] = {dim, size, a.cache.kv_heads, a.cache.pages};
  const cuuint64_t strides[3] = {dim * sizeof(T), size * dim * sizeof(T), a.cache.kv_heads * size * dim * sizeof(T)};
  const cuuint32_t box[4] = {128 / sizeof(T), (cuuint32_t)std::min<cuuint64_t>(size, tile_keys), 1, 1};
  maps->k_step = maps->v_step = 1;
  uint32_t st = encode_map(&maps->k, Format<T>::kMap, 4, a.cache.k, dims, strides, box);
  if (!st) st = encode_map(&maps->v, Format<T>::kMap, 4, a.cache.v, dims, strides, box);
  return st;
}

// Packed keys and values: (element, row, head), boxes of 64 elements of a tile's rows.
template <class T>
uint32_t rows_maps(const AttnArgs& a, uint32_t head_dim, uint32_t tile_keys, Maps* maps) {
  auto one = [&](const pb_rows& r, CUtensorMap* map, uint32_t* step) {
    const bool alone = a.kv_heads == 1 || r.head_stride == 0;
    const cuuint64_t dims[3] = {head_dim, std::max(1u, a.kv_rows), alone ? 1 : a.kv_heads};
    const cuuint64_t strides[2] = {std::max<cuuint64_t>(16, r.row_stride * 2), alone ? 16 : r.head_stride * 2};
    const cuuint32_t box[3] = {64, tile_keys, 1};
    *step = r.head_stride != 0;
    return encode_map(map, Format<T>::kMap, 3, r.data, dims, strides, box);
  };
  uint32_t st = one(a.k, &maps->k, &maps->k_step);
  if (!st) st = one(a.v, &maps->v, &maps->v_step);
  return st;
}

}  // namespace paged
}  // namespace pb
