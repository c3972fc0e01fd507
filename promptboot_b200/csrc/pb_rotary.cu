// Rotary positions with scaled frequencies, in place or beside, and their fused
// form that writes the turned keys and the values to the paged cache.
#include "pb_common.cuh"
#include "pb_paged.cuh"

#include <algorithm>
#include <cmath>
#include <new>

struct pb_rotary {
  pb_rotary_config config;
  float magnitude;
  double turns[128];  // f_i / (2 pi): turns per position of pair i
};

namespace pb {
namespace {

using paged::CacheView;
using paged::Elements;

constexpr int kThreads = 256;
constexpr int kMaxRows = 4;  // rows of one CTA: 58 us where 8 took 63 (16421 rows of 40 heads of 128)

struct RotaryArgs {
  double turns[128];
  const uint32_t* positions;
  const uint32_t* slots;  // NULL: no cache
  pb_rows q, q_out, k, k_out, v;
  CacheView cache;
  uint32_t rows, q_heads, k_heads, v_heads;
  int head_dim, half, rows_per_cta;
  float magnitude;
};

// One CTA turns up to kMaxRows rows.  The cosines and sines of a row are formed
// once for all its heads: the angle in turns as a binary64 product less its
// nearest whole number, so that far positions keep their fraction, then one
// binary32 sincospi.  The heads then stream through as items of two 16-byte words
// (the two words whose elements pair up, or two neighbours where pairs are
// adjacent), consecutive threads on consecutive words of a head.  Bound by
// memory: each element is read and written once.
template <class T, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int V = Elements<T>::n;
  __shared__ float2 turn[kMaxRows][128];
  __shared__ uint32_t pos[kMaxRows], slot[kMaxRows];
  const uint32_t row0 = blockIdx.x * (uint32_t)a.rows_per_cta;
  const int nrows = (int)min((uint32_t)a.rows_per_cta, a.rows - row0);
  if (threadIdx.x < nrows) {
    pos[threadIdx.x] = a.positions[row0 + threadIdx.x];
    slot[threadIdx.x] = a.slots ? a.slots[row0 + threadIdx.x] : PB_NONE;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * a.half; i += kThreads) {
    const int r = i / a.half, p = i - r * a.half;
    const double t = (double)pos[r] * a.turns[p];
    float s, c;
    sincospif((float)(2.0 * (t - rint(t))), &s, &c);
    turn[r][p] = make_float2(__fmul_rn(c, a.magnitude), __fmul_rn(s, a.magnitude));
  }
  __syncthreads();

  const int words = a.head_dim / (2 * V);  // items of a head
  const int heads = (int)(a.q_heads + a.k_heads + a.v_heads);
  const int lane = threadIdx.x % words, step = kThreads / words;
  int head = threadIdx.x / words, r = 0;
  if (head >= step) return;  // the threads past a whole number of heads
  const int turned = a.half / V;  // items that turn (two words each)
  // the two words of this thread's item
  const bool turns = lane < turned;
  const int w0 = turns && !kInterleaved ? lane : 2 * lane;
  const int w1 = turns && !kInterleaved ? lane + turned : 2 * lane + 1;
  for (;;) {
    while (head >= heads) {
      head -= heads;
      if (++r >= nrows) return;
    }
    const bool is_q = head < (int)a.q_heads;
    const bool is_v = head >= (int)(a.q_heads + a.k_heads);
    const uint32_t h = is_q ? head : is_v ? head - a.q_heads - a.k_heads : head - a.q_heads;
    const uint64_t row = row0 + r;
    T* out;
    const pb_rows& in = is_q ? a.q : is_v ? a.v : a.k;
    bool live = pos[r] != PB_NONE;
    if (is_q || !a.slots) {
      const pb_rows& o = is_q ? a.q_out : a.k_out;
      out = static_cast<T*>(o.data) + row * o.row_stride + h * o.head_stride;
    } else {
      const uint32_t s = slot[r], page = s / a.cache.page_size;
      live = live && page < a.cache.pages;
      out = reinterpret_cast<T*>(is_v ? a.cache.v : a.cache.k) +
            (((uint64_t)page * a.cache.kv_heads + h) * a.cache.page_size + s % a.cache.page_size) *
                a.head_dim;
    }
    if (live) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(in.data) +
                                                        row * in.row_stride + h * in.head_stride);
      uint4 u0 = src[w0], u1 = src[w1];
      if (turns && !is_v) {
        float x[V], y[V];
        Elements<T>::load(u0, x);
        Elements<T>::load(u1, y);
        const float2* t = turn[r] + lane * V;
        if (kInterleaved) {
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const float2 c0 = t[i / 2], c1 = t[(V + i) / 2];
            const float b0 = x[i], d0 = y[i];
            x[i] = __fmaf_rn(b0, c0.x, -__fmul_rn(x[i + 1], c0.y));
            x[i + 1] = __fmaf_rn(x[i + 1], c0.x, __fmul_rn(b0, c0.y));
            y[i] = __fmaf_rn(d0, c1.x, -__fmul_rn(y[i + 1], c1.y));
            y[i + 1] = __fmaf_rn(y[i + 1], c1.x, __fmul_rn(d0, c1.y));
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 c = t[i];
            const float b = x[i];
            x[i] = __fmaf_rn(b, c.x, -__fmul_rn(y[i], c.y));
            y[i] = __fmaf_rn(y[i], c.x, __fmul_rn(b, c.y));
          }
        }
        u0 = Elements<T>::store(x);
        u1 = Elements<T>::store(y);
      }
      uint4* dst = reinterpret_cast<uint4*>(out);
      dst[w0] = u0;
      dst[w1] = u1;
    }
    head += step;
  }
}

template <class T>
uint32_t launch_rotary(RotaryArgs& a, uint32_t layout, cudaStream_t s) {
  // Enough CTAs for every SM first; then more rows per CTA.
  a.rows_per_cta = (int)std::min<uint32_t>(kMaxRows, std::max<uint32_t>(1, a.rows / (148 * 4)));
  const uint32_t grid = (a.rows + a.rows_per_cta - 1) / a.rows_per_cta;
  if (layout == PB_ROTARY_INTERLEAVED) rotary_kernel<T, true><<<grid, kThreads, 0, s>>>(a);
  else rotary_kernel<T, false><<<grid, kThreads, 0, s>>>(a);
  PB_CUDA(cudaGetLastError());
  return PB_OK;
}

uint32_t run_rotary(const pb_rotary* rotary, RotaryArgs& a, uint32_t type, cudaStream_t s) {
  std::copy(rotary->turns, rotary->turns + 128, a.turns);
  a.magnitude = rotary->magnitude;
  a.head_dim = (int)rotary->config.head_dim;
  a.half = (int)rotary->config.rotary_dim / 2;
  const uint32_t layout = rotary->config.layout;
  if (type == PB_TYPE_F32) return launch_rotary<float>(a, layout, s);
  if (type == PB_TYPE_F16) return launch_rotary<__half>(a, layout, s);
  return launch_rotary<__nv_bfloat16>(a, layout, s);
}

// An output that is its input has to be all of it: same data, same strides.
bool same_or_apart(const pb_rows* in, const pb_rows* out) {
  return in->data != out->data ||
         (in->row_stride == out->row_stride && in->head_stride == out->head_stride);
}

}  // namespace
}  // namespace pb

extern "C" {

uint32_t pb_rotary_create(const pb_rotary_config* c, pb_rotary** out) {
  const char* who = "pb_rotary_create";
  if (!c || !out) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  *out = nullptr;
  if (!c->head_dim || c->head_dim % 16 || c->head_dim > 256 || !c->rotary_dim ||
      c->rotary_dim % 16 || c->rotary_dim > c->head_dim)
    return pb::paged::refuse(PB_CAPACITY, who,
                             "head_dim and rotary_dim must be multiples of 16, rotary_dim <= head_dim <= 256");
  if (c->layout > PB_ROTARY_INTERLEAVED || c->scaling > PB_SCALING_YARN)
    return pb::paged::refuse(PB_CAPACITY, who, "unknown layout or scaling");
  const bool scaled = c->scaling != PB_SCALING_NONE;
  const bool spans = c->scaling == PB_SCALING_BANDS || c->scaling == PB_SCALING_YARN;
  if (!(c->theta > 1.0) || !std::isfinite(c->theta) || !(c->magnitude >= 0.0) ||
      !std::isfinite(c->magnitude))
    return pb::paged::refuse(PB_CAPACITY, who, "theta must be above 1 and magnitude not negative, both finite");
  if (scaled && (!(c->factor >= 1.0) || !std::isfinite(c->factor)))
    return pb::paged::refuse(PB_CAPACITY, who, "factor must be 1 or more and finite");
  double low = c->low, high = c->high;
  if (low == 0.0 && high == 0.0) {
    low = 1.0;
    high = c->scaling == PB_SCALING_YARN ? 32.0 : 4.0;
  }
  if (spans && (!(c->original >= 1.0) || !std::isfinite(c->original) || !(low > 0.0) ||
                !(high > low) || !std::isfinite(high)))
    return pb::paged::refuse(PB_CAPACITY, who, "original must be 1 or more and 0 < low < high, all finite");
  pb_rotary* r = new (std::nothrow) pb_rotary();
  if (!r) return pb::paged::refuse(PB_CAPACITY, who, "out of host memory");
  r->config = *c;
  const double two_pi = 6.283185307179586476925;
  const int dim = (int)c->rotary_dim, half = dim / 2;
  double i0 = 0.0, i1 = 1.0;
  if (c->scaling == PB_SCALING_YARN) {
    auto place = [&](double t) {
      return dim * std::log(c->original / (two_pi * t)) / (2.0 * std::log(c->theta));
    };
    i0 = std::min(std::max(std::floor(place(high)), 0.0), dim - 1.0);
    i1 = std::min(std::max(std::ceil(place(low)), 0.0), dim - 1.0);
    if (!(i1 > i0)) i1 = i0 + 0.001;
  }
  for (int i = 0; i < half; ++i) {
    const double f = std::pow(c->theta, -(double)i / half);
    double keep = 1.0;  // share of the unscaled frequency
    if (c->scaling == PB_SCALING_LINEAR) keep = 0.0;
    if (c->scaling == PB_SCALING_BANDS) keep = (c->original * f / two_pi - low) / (high - low);
    if (c->scaling == PB_SCALING_YARN) keep = 1.0 - (i - i0) / (i1 - i0);
    keep = std::min(std::max(keep, 0.0), 1.0);
    r->turns[i] = (scaled ? f / c->factor * (1.0 - keep) + f * keep : f) / two_pi;
  }
  r->magnitude = (float)(c->magnitude > 0.0                  ? c->magnitude
                         : c->scaling == PB_SCALING_YARN ? 0.1 * std::log(c->factor) + 1.0
                                                         : 1.0);
  *out = r;
  return PB_OK;
}

void pb_rotary_destroy(pb_rotary* rotary) { delete rotary; }

uint32_t pb_rotary_device(const pb_rotary* rotary, uint32_t type, uint32_t rows,
                          const uint32_t* positions, uint32_t q_heads, const pb_rows* q,
                          const pb_rows* q_out, uint32_t k_heads, const pb_rows* k,
                          const pb_rows* k_out, void* stream) {
  const char* who = "pb_rotary_device";
  const uint32_t bytes = pb::paged::type_bytes(type);
  if (!rotary || !positions) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  if (!bytes) return pb::paged::refuse(PB_CAPACITY, who, "unknown element type");
  if (!rows || rows > 1u << 30 || !q_heads || q_heads > 1024 || k_heads > 1024)
    return pb::paged::refuse(PB_CAPACITY, who, "rows, q_heads or k_heads out of range");
  uint32_t st;
  if ((st = pb::paged::check_rows(q, bytes, who, "q"))) return st;
  if ((st = pb::paged::check_output(q_out, bytes, rows, q_heads, who, "q_out"))) return st;
  if (k_heads && (st = pb::paged::check_rows(k, bytes, who, "k"))) return st;
  if (k_heads && (st = pb::paged::check_output(k_out, bytes, rows, k_heads, who, "k_out"))) return st;
  if (!pb::same_or_apart(q, q_out) || (k_heads && !pb::same_or_apart(k, k_out)))
    return pb::paged::refuse(PB_CAPACITY, who, "an output in place needs its input's strides");
  pb::RotaryArgs a{};
  a.positions = positions;
  a.rows = rows; a.q_heads = q_heads; a.k_heads = k_heads;
  a.q = *q; a.q_out = *q_out;
  if (k_heads) { a.k = *k; a.k_out = *k_out; }
  return pb::run_rotary(rotary, a, type, (cudaStream_t)stream);
}

uint32_t pb_rotary_cache_device(const pb_rotary* rotary, uint32_t rows, const uint32_t* positions,
                                uint32_t q_heads, const pb_rows* q, const pb_rows* q_out,
                                const pb_rows* k, const pb_rows* v, const pb_cache* cache,
                                uint32_t layer, const uint32_t* slots, void* stream) {
  const char* who = "pb_rotary_cache_device";
  if (!rotary || !positions || !slots) return pb::paged::refuse(PB_CAPACITY, who, "a NULL argument");
  uint32_t st;
  if ((st = pb::paged::check_cache(cache, who))) return st;
  const uint32_t bytes = pb::paged::type_bytes(cache->type);
  if (!rows || rows > 1u << 30 || !q_heads || q_heads > 1024)
    return pb::paged::refuse(PB_CAPACITY, who, "rows or q_heads out of range");
  if (layer >= cache->layers) return pb::paged::refuse(PB_CAPACITY, who, "no such layer");
  if (cache->head_dim != rotary->config.head_dim)
    return pb::paged::refuse(PB_CAPACITY, who, "the cache has another head_dim");
  if ((st = pb::paged::check_rows(q, bytes, who, "q"))) return st;
  if ((st = pb::paged::check_output(q_out, bytes, rows, q_heads, who, "q_out"))) return st;
  if ((st = pb::paged::check_rows(k, bytes, who, "k"))) return st;
  if ((st = pb::paged::check_rows(v, bytes, who, "v"))) return st;
  if (!pb::same_or_apart(q, q_out))
    return pb::paged::refuse(PB_CAPACITY, who, "an output in place needs its input's strides");
  pb::RotaryArgs a{};
  a.positions = positions; a.slots = slots;
  a.rows = rows; a.q_heads = q_heads; a.k_heads = a.v_heads = cache->kv_heads;
  a.q = *q; a.q_out = *q_out; a.k = *k; a.v = *v;
  a.cache = pb::paged::layer_view(cache, layer);
  return pb::run_rotary(rotary, a, cache->type, (cudaStream_t)stream);
}

}  // extern "C"
