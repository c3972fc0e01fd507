// Shared by the paged serving operators: argument checks, element types, and the
// device view of rows and of the paged cache.
#pragma once

#include "pb_host.h"

#include <cstdio>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace pb {
namespace paged {

inline uint32_t refuse(uint32_t status, const char* who, const char* what) {
  char text[256];
  std::snprintf(text, sizeof text, "%s: %s", who, what);
  set_last_error(text);
  return status;
}

inline uint32_t type_bytes(uint32_t type) {
  return type == PB_TYPE_F32 ? 4u : type == PB_TYPE_F16 || type == PB_TYPE_BF16 ? 2u : 0u;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// A pb_rows operand: 16-byte aligned data and strides.
inline uint32_t check_rows(const pb_rows* r, uint32_t bytes, const char* who, const char* name) {
  char text[160];
  if (!r || !r->data) {
    std::snprintf(text, sizeof text, "%s is NULL", name);
    return refuse(PB_CAPACITY, who, text);
  }
  if (!aligned16(r->data) || (r->row_stride * bytes) % 16 || (r->head_stride * bytes) % 16) {
    std::snprintf(text, sizeof text, "%s needs 16-byte aligned data, row stride and head stride", name);
    return refuse(PB_ALIGNMENT, who, text);
  }
  return PB_OK;
}

// A pb_rows that is written: its rows and heads may not lie on one another (a stride of 0).
inline uint32_t check_output(const pb_rows* r, uint32_t bytes, uint32_t rows, uint32_t heads, const char* who,
                             const char* name) {
  const uint32_t st = check_rows(r, bytes, who, name);
  if (st) return st;
  if ((rows > 1 && !r->row_stride) || (heads > 1 && !r->head_stride)) {
    char text[160];
    std::snprintf(text, sizeof text, "%s needs a row stride and a head stride", name);
    return refuse(PB_CAPACITY, who, text);
  }
  return PB_OK;
}

inline uint32_t check_cache(const pb_cache* c, const char* who) {
  if (!c || !c->k || !c->v) return refuse(PB_CAPACITY, who, "the cache is NULL");
  const uint32_t bytes = type_bytes(c->type);
  if (!bytes) return refuse(PB_CAPACITY, who, "unknown element type");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return refuse(PB_CAPACITY, who, "page_size must be 16, 32, 64, 128 or 256");
  if (!c->layers || !c->pages || !c->kv_heads || c->kv_heads > 1024)
    return refuse(PB_CAPACITY, who, "the cache needs layers, pages and 1 to 1024 heads");
  if ((uint64_t)c->pages * c->page_size >= 1ull << 31)
    return refuse(PB_CAPACITY, who, "pages * page_size must stay below 2^31");
  if (!c->head_dim || c->head_dim % 16 || c->head_dim > 256)
    return refuse(PB_CAPACITY, who, "head_dim must be a multiple of 16 up to 256");
  if (!aligned16(c->k) || !aligned16(c->v) || (c->layer_stride * bytes) % 16)
    return refuse(PB_ALIGNMENT, who, "the cache needs 16-byte aligned data and layer stride");
  if (c->layers > 1 &&
      c->layer_stride < (uint64_t)c->pages * c->kv_heads * c->page_size * c->head_dim)
    return refuse(PB_CAPACITY, who, "layer_stride is smaller than a layer's pages");
  return PB_OK;
}

// One layer of a cache, as kernels see it.
struct CacheView {
  uint8_t *k, *v;
  uint32_t pages, page_size, kv_heads, head_dim;
};

inline CacheView layer_view(const pb_cache* c, uint32_t layer) {
  const uint64_t at = (uint64_t)layer * c->layer_stride * type_bytes(c->type);
  return {static_cast<uint8_t*>(c->k) + at, static_cast<uint8_t*>(c->v) + at, c->pages,
          c->page_size, c->kv_heads, c->head_dim};
}

// 16 bytes of elements as binary32 and back (one rounding, to nearest even).
template <class T>
struct Elements;
template <>
struct Elements<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void load(uint4 w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y);
    x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 store(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                      __float_as_uint(x[3]));
  }
};
template <>
struct Elements<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void load(uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2_raw r;
      r.x = (unsigned short)u[i];
      r.y = (unsigned short)(u[i] >> 16);
      const float2 f = __half22float2(__half2(r));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ uint4 store(const float (&x)[8]) {
    return make_uint4(pair(x[0], x[1]), pair(x[2], x[3]), pair(x[4], x[5]), pair(x[6], x[7]));
  }
};
template <>
struct Elements<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void load(uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ uint4 store(const float (&x)[8]) {
    return make_uint4(pair(x[0], x[1]), pair(x[2], x[3]), pair(x[4], x[5]), pair(x[6], x[7]));
  }
};

}  // namespace paged
}  // namespace pb
