// Paged serving attention of binary32 elements on the CUDA cores, with every product
// and sum in binary32.
//
// One pass over the keys per row with a running maximum m and sum l (Milakov and
// Gimelshein's online softmax): for a tile of scores x (in powers of two),
//   m' = max(m, max x),  o <- o 2^(m - m') + sum 2^(x - m') v,  l alike,
// and out = o / l.
//
// The keys of the next tile are on their way while the weights are found and the values
// added, its values while its scores are.  Bound by the latency of a warp's chain and
// the reads of shared memory that feed its multiply-adds.  Row tiles of 32, four CTAs an
// SM (three of prompts at heads of 128, by their registers): a prompt of 2500 tokens, 14 heads of 64 to 2, takes 370 us, 30 TFLOP/s (tiles of 64:
// 394, of 16: 492); 8 of 2500 in all 112 (139, 126); trees of 8 nodes over 32 x 3000
// positions, 32 heads of 128 to 8, 438 us, 23 TFLOP/s (886 with tiles of 64, half empty).
#include "pb_attention_launch.h"

namespace pb {
namespace paged {
namespace {

constexpr int kThreads = 128;
constexpr int kLeast = 2;  // key tiles of a CTA's run at least

// kRpt rows and kKpt keys per thread: 8 thread rows x 16 thread columns.
template <int kDim, int kRpt>
struct Simt {
  static constexpr int kRows = 8 * kRpt;
  static constexpr int kKeys = kDim == 64 ? 64 : 32;
  static constexpr int kKpt = kKeys / 16;
  static constexpr int kPad = kDim + 4;   // row pitch: 16-byte reads of 8 rows hit all banks once
  static constexpr int kPadP = kKeys + 4;
  static constexpr int kCtas = 4;        // per SM, by shared memory for row tiles of 32
  static constexpr int kWords = kRows * kPad + 2 * kKeys * kPad + kRows * kPadP;
  static size_t bytes(uint32_t seqs) { return (size_t)(kWords + seqs) * 4; }
};

// Four elements at `dst` from `src` (zeros: NULL).
__device__ __forceinline__ void fill(float* dst, const float* src) {
  *reinterpret_cast<float4*>(dst) =
      src ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
}

// The same on its way, 16 bytes; `any` is some valid address.
__device__ __forceinline__ void copy16(float* dst, const float* src, const void* any) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src ? src : any), "r"(src ? 16 : 0)
               : "memory");
}
// Waits until at most the newest group of this thread's copies is under way.
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

template <int kDim, int kRpt, bool kTree>
__global__ void __launch_bounds__(kThreads, kTree ? Simt<kDim, kRpt>::kCtas : 1) attention_simt_kernel(const __grid_constant__ AttnArgs a) {
  using C = Simt<kDim, kRpt>;
  constexpr int kRows = C::kRows, kKeys = C::kKeys, kKpt = C::kKpt, kCols = kDim / 64;
  extern __shared__ __align__(16) float smem[];
  float* qs = smem;
  float* ks = qs + kRows * C::kPad;
  float* vs = ks + kKeys * C::kPad;
  float* ps = vs + kKeys * C::kPad;
  if (kTree) pdl_trigger();
  uint32_t* prefix = reinterpret_cast<uint32_t*>(ps + kRows * C::kPadP);
  work_prefix<kTree, kRows, kKeys, kThreads>(a, prefix);
  const uint32_t total = prefix[a.seqs - 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const uint32_t page_bits = kTree ? 31 - __clz((int)a.cache.page_size) : 0;  // a power of two

  uint32_t next, end;  // this CTA's items: one segment, or a run of key tiles
  if (kTree) {
    const Share<kLeast> share(total, gridDim.x);
    if (threadIdx.x == kThreads - 1) note_join<kRows, kKeys>(a, prefix, share, blockIdx.x);
    if (total == 0) return;
    if (blockIdx.x >= share.runs) return;
    next = share.start(blockIdx.x);
    end = share.start(blockIdx.x + 1);
  } else {
    if (blockIdx.x >= total) return;
    next = blockIdx.x;
    end = next + 1;
  }

  while (next < end) {
    Piece p;
    Sequence s;
    uint32_t rows;
    take_piece<kTree, kRows, kKeys>(a, prefix, blockIdx.x, next, end, p, s, rows);
    __syncthreads();  // the piece before is done with shared memory
    constexpr int kWords = kDim / 4;
#pragma unroll 2
    for (int i = threadIdx.x; i < kRows * kWords; i += kThreads) {
      const int r = i / kWords, c = i % kWords * 4;
      const uint32_t row = p.row_tile * kRows + r;
      const float* src = nullptr;
      if (row < rows)
        src = static_cast<const float*>(a.q.data) + (uint64_t)(s.q0 + row / a.group) * a.q.row_stride +
              (uint64_t)(p.head * a.group + row % a.group) * a.q.head_stride + c;
      fill(qs + r * C::kPad + c, src);
    }
    RowView view[kRpt];
    uint32_t all_see = 0xffffffffu;  // keys that every row of this thread sees
#pragma unroll
    for (int i = 0; i < kRpt; ++i) {
      const uint32_t row = p.row_tile * kRows + ty + 8 * i;
      view[i] = row < rows ? row_view<kTree>(a, s, row / a.group) : RowView{0xffffffffu, 0ull};
      all_see = min(all_see, view[i].all);
    }
    float m[kRpt], l[kRpt];
    float4 o[kRpt][kCols];
#pragma unroll
    for (int i = 0; i < kRpt; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }

    // Copies tile `tile` of the keys or the values on its way; zeros where there are none.
    auto send = [&](float* to, bool values, uint32_t tile) {
      if (tile < p.tile1) {
        const pb_rows& packed = values ? a.v : a.k;
        const float* cached = reinterpret_cast<const float*>(values ? a.cache.v : a.cache.k);
#pragma unroll 4
        for (int i = threadIdx.x; i < kKeys * kWords; i += kThreads) {
          const int j = i / kWords, c = i % kWords * 4;
          const uint32_t key = tile * kKeys + j;
          const float* from = nullptr;
          if (key < s.len) {
            if (kTree) {
              const uint32_t page = a.tables[(uint64_t)p.seq * a.table_width + (key >> page_bits)];
              if (page < a.cache.pages)
                from = cached + ((((uint64_t)page * a.cache.kv_heads + p.head) << page_bits) +
                                 (key & (a.cache.page_size - 1))) * kDim + c;
            } else {
              from = static_cast<const float*>(packed.data) + (uint64_t)(s.kv0 + key) * packed.row_stride +
                     p.head * packed.head_stride + c;
            }
          }
          copy16(to + j * C::kPad + c, from, a.q.data);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    send(ks, false, p.tile0);
    send(vs, true, p.tile0);
    for (uint32_t tile = p.tile0; tile < p.tile1; ++tile) {
      const uint32_t key0 = tile * kKeys;
      copies_wait();  // the keys
      __syncthreads();

      float sc[kRpt][kKpt];  // key tx + 16 j
#pragma unroll
      for (int i = 0; i < kRpt; ++i)
#pragma unroll
        for (int j = 0; j < kKpt; ++j) sc[i][j] = 0.f;
#pragma unroll 4
      for (int c = 0; c < kDim; c += 4) {
        float4 kf[kKpt];
#pragma unroll
        for (int j = 0; j < kKpt; ++j)
          kf[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * C::kPad + c);
#pragma unroll
        for (int i = 0; i < kRpt; ++i) {
          const float4 qf = *reinterpret_cast<const float4*>(qs + (ty + 8 * i) * C::kPad + c);
#pragma unroll
          for (int j = 0; j < kKpt; ++j) {
            sc[i][j] = __fmaf_rn(qf.x, kf[j].x, sc[i][j]);
            sc[i][j] = __fmaf_rn(qf.y, kf[j].y, sc[i][j]);
            sc[i][j] = __fmaf_rn(qf.z, kf[j].z, sc[i][j]);
            sc[i][j] = __fmaf_rn(qf.w, kf[j].w, sc[i][j]);
          }
        }
      }
      __syncthreads();
      send(ks, false, tile + 1);
      // A key that a row does not see gets the weight -0, which the sums below tell
      // from the weight +0 of a score far below the maximum: its value is left out
      // whatever it holds.
      const bool masked = key0 + kKeys > all_see;
#pragma unroll
      for (int i = 0; i < kRpt; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kKpt; ++j) {
          const bool seen = !masked || view[i].sees(key0 + tx + 16 * j);
          sc[i][j] = seen ? __fmul_rn(sc[i][j], a.scale_log2) : -INFINITY;
          top = max_nan(top, sc[i][j], -INFINITY);
        }
#pragma unroll
        for (int d = 8; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d), -INFINITY);
        // Not a number where a score is not: then so are the row and what a join takes of it.
        const float to = max_nan(m[i], top, -INFINITY);
        const float base = to == -INFINITY ? 0.f : to;
        const float keep = exp2f(m[i] - base);  // 0 from -inf
        m[i] = to;
        l[i] = __fmul_rn(l[i], keep);
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          o[i][c].x = __fmul_rn(o[i][c].x, keep); o[i][c].y = __fmul_rn(o[i][c].y, keep);
          o[i][c].z = __fmul_rn(o[i][c].z, keep); o[i][c].w = __fmul_rn(o[i][c].w, keep);
        }
#pragma unroll
        for (int j = 0; j < kKpt; ++j) {
          const bool seen = !masked || view[i].sees(key0 + tx + 16 * j);
          const float w = seen ? exp2f(__fsub_rn(sc[i][j], base)) : -0.f;
          l[i] += seen ? w : 0.f;
          ps[(ty + 8 * i) * C::kPadP + tx + 16 * j] = w;
        }
      }
      copies_wait();    // the values
      __syncthreads();  // (a row's weights come from lanes of its warp alone)
      auto add_values = [&](auto checked) {
#pragma unroll 2
        for (int j = 0; j < kKeys; j += 4) {
          float4 vf[4][kCols];
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < kCols; ++c)
              vf[u][c] = *reinterpret_cast<const float4*>(vs + (j + u) * C::kPad + c * 64 + tx * 4);
#pragma unroll
          for (int i = 0; i < kRpt; ++i) {
            const float4 w4 = *reinterpret_cast<const float4*>(ps + (ty + 8 * i) * C::kPadP + j);
            const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              if (decltype(checked)::value && __float_as_uint(w[u]) == 0x80000000u) continue;
#pragma unroll
              for (int c = 0; c < kCols; ++c) {
                o[i][c].x = __fmaf_rn(w[u], vf[u][c].x, o[i][c].x);
                o[i][c].y = __fmaf_rn(w[u], vf[u][c].y, o[i][c].y);
                o[i][c].z = __fmaf_rn(w[u], vf[u][c].z, o[i][c].z);
                o[i][c].w = __fmaf_rn(w[u], vf[u][c].w, o[i][c].w);
              }
            }
          }
        }
      };
      if (masked) add_values(std::true_type{});
      else add_values(std::false_type{});
      __syncthreads();
      send(vs, true, tile + 1);
    }

#pragma unroll
    for (int i = 0; i < kRpt; ++i) {
#pragma unroll
      for (int d = 8; d; d >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
      const uint32_t r = ty + 8 * i, row = p.row_tile * kRows + r;
      if (row >= rows) continue;
      if (p.partial >= 0) {
        float* rec = a.partial + (size_t)p.partial * partial_words<kRows, kDim>();
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          *reinterpret_cast<float4*>(rec + r * kDim + c * 64 + tx * 4) = o[i][c];
        if (tx == 0) {
          rec[kRows * kDim + r] = m[i];
          rec[kRows * kDim + kRows + r] = l[i];
        }
      } else {
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        float* out = static_cast<float*>(a.out.data) + (uint64_t)(s.q0 + row / a.group) * a.out.row_stride +
                 (uint64_t)(p.head * a.group + row % a.group) * a.out.head_stride;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          store4(out + c * 64 + tx * 4,
                 make_float4(o[i][c].x * inv, o[i][c].y * inv, o[i][c].z * inv, o[i][c].w * inv));
      }
    }
  }
}

template <int kDim, int kRpt, bool kTree>
uint32_t launch(AttnArgs a, uint32_t grid, cudaStream_t s) {
  using C = Simt<kDim, kRpt>;
  auto kernel = attention_simt_kernel<kDim, kRpt, kTree>;
  static std::atomic<uint64_t> configured{0};
  if (attribute_needed(configured)) {
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)C::bytes(PB_MAX_SEQS)));
    attribute_done(configured);
  }
  if (kTree) place_workspace(a, grid, C::kRows, kDim);
  kernel<<<grid, kThreads, C::bytes(a.seqs), s>>>(a);
  PB_CUDA(cudaGetLastError());
  return kTree ? launch_combine<float, kDim, C::kRows>(a, grid, s) : PB_OK;
}

constexpr int kTreeCtas = Simt<64, 4>::kCtas;
constexpr int kFewRpt = 2, kManyRpt = 4;  // 16 or 32 rows of a tile

}  // namespace

uint32_t simt_prompt(const AttnArgs& a, uint32_t head_dim, cudaStream_t s) {
  const uint32_t rows = a.q_rows * a.group;
  // Row tiles of 16 where there are no more than some two tiles of 32 to an SM.
  const bool small = (uint64_t)rows * a.kv_heads < 64ull * tree_ctas(1);
  const uint32_t grid = (rows / (small ? 8 * kFewRpt : 8 * kManyRpt) + a.seqs) * a.kv_heads;
  if (small)
    return head_dim == 64 ? launch<64, kFewRpt, false>(a, grid, s) : launch<128, kFewRpt, false>(a, grid, s);
  return head_dim == 64 ? launch<64, kManyRpt, false>(a, grid, s) : launch<128, kManyRpt, false>(a, grid, s);
}

uint64_t simt_tree_words(uint32_t head_dim) { return tree_words(tree_ctas(kTreeCtas), 8 * kManyRpt, head_dim); }

uint32_t simt_tree(const AttnArgs& a, uint32_t head_dim, cudaStream_t s) {
  const uint32_t grid = tree_ctas(kTreeCtas);
  return head_dim == 64 ? launch<64, kManyRpt, true>(a, grid, s) : launch<128, kManyRpt, true>(a, grid, s);
}

}  // namespace paged
}  // namespace pb
