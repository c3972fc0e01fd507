// Tree attention of few rows per sequence and key head (16-bit types): single
// tokens and small drafts, where the keys and values are read once from memory and
// little is computed on them.
//
// At most 32 rows against tiles of 8 KB of keys and values: each warp walks a run of
// tiles of its own through a ring of its own, filled by TMA (128-byte swizzle) that it
// issues itself, and runs the online softmax of pb_attention_simt.cu on mma.sync
// m16n8k16 products, whose accumulators are the next product's operand as they stand.
// Warps of a CTA share nothing, so that one's segment ends under the others' tiles (four
// warps to a run, joined at each segment's end, took 44 us with its join where this takes
// 37.6, for 256 single tokens over 512 to 1535 positions).  The legacy tensor path is the right one here: a tcgen05 tile has 128 rows, so that one
// token of seven heads would pay for 18 times its products, and its scores would pass
// through TMEM on the way.  Bound by memory and by the latency of a warp's chain
// through a tile (some 1000 cycles), of which twelve are under way on an SM at heads of 64
// with one row group and eight else; one warp that fed all others was a bound of its own
// (a copy takes it some 100 cycles).
#include "pb_attention_launch.h"
#include "pb_attention_tma.cuh"

namespace pb {
namespace paged {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kLeast = 4;

// kTiles row groups of 16.
template <int kDim, int kTiles>
struct Few {
  static constexpr int kKeys = kDim == 64 ? 32 : 16;    // of a tile
  static constexpr int kRows = 16 * kTiles;
  static constexpr int kCtas = kDim == 64 && kTiles == 1 ? 3 : 2;  // per SM, by registers
  static constexpr int kStages = kCtas == 3 ? 2 : 3;    // of a warp
  static constexpr int kHalves = kDim / 64;
  static constexpr int kBlock = kKeys * 128;
  static constexpr int kTile = kHalves * kBlock;        // K or V
  static constexpr int kBarOff = kWarps * kStages * 2 * kTile;
  static constexpr int kPrefixOff = kBarOff + kWarps * kStages * 8 + 16;
  static size_t bytes(uint32_t seqs) { return 1024 + kPrefixOff + (size_t)seqs * 4; }
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <class T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class T, int kDim, int kTiles>
__global__ void __launch_bounds__(kThreads, Few<kDim, kTiles>::kCtas)
attention_few_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Maps maps) {
  using C = Few<kDim, kTiles>;
  using F = Format<T>;
  constexpr int kRows = C::kRows, kKeys = C::kKeys, kStages = C::kStages, kHalves = C::kHalves;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kWarps * kStages);
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + C::kPrefixOff);

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(&bars[i], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  work_prefix<true, kRows, kKeys, kThreads>(a, prefix);  // ends with a barrier of the block
  const uint32_t total = prefix[a.seqs - 1];
  const Share<kLeast> share(total, gridDim.x * kWarps);
  const uint32_t run = blockIdx.x * kWarps + warp;
  uint32_t next = run < share.runs ? share.start(run) : total;
  const uint32_t end = run < share.runs ? share.start(run + 1) : total;

  TileRing<T, kRows, kKeys, kHalves, kStages> ring(a, maps, prefix, bars + warp * kStages,
                                                   smem + warp * kStages * 2 * C::kTile, next, end);
  if (lane == 0) note_join<kRows, kKeys>(a, prefix, share, run);

  const int r0 = lane >> 2, c0 = (lane & 3) * 2;  // this thread's fragment row (and + 8) and column
  Sequence s;
  uint32_t rows;
  int used = 0;  // tiles
  bool stop = false;
  while (next < end && !stop) {
    Piece p;
    take_piece<true, kRows, kKeys>(a, prefix, run, next, end, p, s, rows);
    bool mend = false;  // a value was taken out
    // Row h % 2 of row group h / 2: the fragment rows r0 and r0 + 8.
    uint32_t row[2 * kTiles];
    RowView view[2 * kTiles];
    uint32_t qf[kTiles][kDim / 16][4];  // Q as the first operand
#pragma unroll
    for (int h = 0; h < 2 * kTiles; ++h) {
      row[h] = p.row_tile * kRows + r0 + 8 * h;
      const bool there = row[h] < rows;
      const uint32_t token = row[h] / a.group;
      // Rows past the last see everything: zeros times finite or other keys, never stored.
      view[h] = there ? row_view<true>(a, s, token) : RowView{0xffffffffu, 0ull};
      const T* src = static_cast<const T*>(a.q.data) + (uint64_t)(s.q0 + token) * a.q.row_stride +
                     (uint64_t)(p.head * a.group + row[h] % a.group) * a.q.head_stride + c0;
#pragma unroll
      for (int k = 0; k < kDim / 16; ++k) {
        qf[h / 2][k][h % 2] = there ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
        qf[h / 2][k][2 + h % 2] = there ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
      }
    }
    float m[2 * kTiles], l[2 * kTiles];
    float o[kTiles][kDim / 8][4];
#pragma unroll
    for (int h = 0; h < 2 * kTiles; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
    }
#pragma unroll
    for (int g = 0; g < kTiles; ++g)
#pragma unroll
      for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[g][i][j] = 0.f;
    const uint32_t mask0 = s.context / kKeys;  // tiles from here on hold a key that some row does not see

    for (uint32_t tile = p.tile0; tile < p.tile1; ++tile) {
      if (!wait_soon(&ring.full[used % kStages], (used / kStages) & 1, abort_flag)) { stop = true; break; }
      uint8_t* tile_keys = ring.keys(used++);
      const uint32_t kt = smem_u32(tile_keys), vt = kt + C::kTile;
      float sc[kTiles][kKeys / 8][4];
#pragma unroll
      for (int g = 0; g < kTiles; ++g)
#pragma unroll
        for (int j = 0; j < kKeys / 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[g][j][i] = 0.f;
#pragma unroll
      for (int k = 0; k < kDim / 16; ++k) {
#pragma unroll
        for (int j = 0; j < kKeys / 16; ++j) {
          const int key = j * 16 + (lane >> 4) * 8 + (lane & 7), chunk = k * 2 + ((lane >> 3) & 1);
          uint32_t b[4];
          ldmatrix4(kt + chunk / 8 * C::kBlock + key * 128 + ((chunk % 8) ^ (key & 7)) * 16, b);
#pragma unroll
          for (int g = 0; g < kTiles; ++g) {
            mma16<T>(sc[g][2 * j], qf[g][k], b[0], b[1]);
            mma16<T>(sc[g][2 * j + 1], qf[g][k], b[2], b[3]);
          }
        }
      }
      const bool masked = tile >= mask0;
      const uint32_t key0 = tile * kKeys;
      if (masked) {
#pragma unroll
        for (int g = 0; g < kTiles; ++g)
#pragma unroll
          for (int j = 0; j < kKeys / 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!view[2 * g + i / 2].sees(key0 + j * 8 + c0 + (i & 1))) sc[g][j][i] = -INFINITY;
      }
      float base[2 * kTiles], keep[2 * kTiles];
      bool moved = false;
#pragma unroll
      for (int h = 0; h < 2 * kTiles; ++h) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kKeys / 8; ++j)
          top = max_nan(top, sc[h / 2][j][h % 2 * 2], sc[h / 2][j][h % 2 * 2 + 1]);
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1), -INFINITY);
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2), -INFINITY);
        top = __fmul_rn(top, a.scale_log2);
        keep[h] = 1.f;
        if (!(top < INFINITY)) {
          m[h] = NAN;  // a score that is not a number or +inf: so is the row
        } else if (m[h] == -INFINITY) {
          m[h] = top;  // nothing has been added yet
        } else if (top > m[h] + F::kSlack) {
          keep[h] = exp2_fast(m[h] - top);
          m[h] = top;
          moved = true;
        }
        base[h] = F::kRaise - (m[h] == -INFINITY ? 0.f : m[h]);
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int h = 0; h < 2 * kTiles; ++h) {
          l[h] = __fmul_rn(l[h], keep[h]);
#pragma unroll
          for (int i = 0; i < kDim / 8; ++i) {
            o[h / 2][i][h % 2 * 2] = __fmul_rn(o[h / 2][i][h % 2 * 2], keep[h]);
            o[h / 2][i][h % 2 * 2 + 1] = __fmul_rn(o[h / 2][i][h % 2 * 2 + 1], keep[h]);
          }
        }
      }
      uint32_t pf[kTiles][kKeys / 16][4];  // P as the first operand
#pragma unroll
      for (int g = 0; g < kTiles; ++g)
#pragma unroll
        for (int j = 0; j < kKeys / 8; ++j) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = exp2_fast(__fmaf_rn(sc[g][j][i], a.scale_log2, base[2 * g + i / 2]));
            l[2 * g + i / 2] += w[i];
          }
          pf[g][j / 2][j % 2 * 2] = Elements<T>::pair(w[0], w[1]);
          pf[g][j / 2][j % 2 * 2 + 1] = Elements<T>::pair(w[2], w[3]);
        }
      if (masked) {
        // The tile's value rows: zero past the keys, and without what is not finite.
        mend |= __any_sync(0xffffffffu, clean_value_row<F, kDim, C::kBlock, 32 / kKeys>(
                                            tile_keys + C::kTile, lane % kKeys, lane / kKeys,
                                            key0 + lane % kKeys >= s.len));
        __syncwarp();  // cleaned rows before other lanes read them (a vote orders no memory)
      }
#pragma unroll
      for (int j = 0; j < kKeys / 16; ++j) {
#pragma unroll
        for (int n = 0; n < kDim / 16; ++n) {
          const int key = j * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), chunk = n * 2 + (lane >> 4);
          uint32_t b[4];
          ldmatrix4_trans(vt + chunk / 8 * C::kBlock + key * 128 + ((chunk % 8) ^ (key & 7)) * 16, b);
#pragma unroll
          for (int g = 0; g < kTiles; ++g) {
            mma16<T>(o[g][2 * n], pf[g][j], b[0], b[1]);
            mma16<T>(o[g][2 * n + 1], pf[g][j], b[2], b[3]);
          }
        }
      }
      if (masked) fence_async_smem();  // cleaned rows before the next copy over them
      __syncwarp();
      ring.send();
    }

    if (stop) break;

    // The piece is done: O / l, or O with its maximum and sum.
#pragma unroll
    for (int h = 0; h < 2 * kTiles; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (row[h] >= rows) continue;
      float y[kDim / 8][2];
#pragma unroll
      for (int i = 0; i < kDim / 8; ++i) {
        y[i][0] = o[h / 2][i][h % 2 * 2];
        y[i][1] = o[h / 2][i][h % 2 * 2 + 1];
      }
      if (mend) {
        // A weight is positive: what is not finite passes through the sum as it is.
        for (uint32_t key = max(p.tile0, mask0) * kKeys; key < min(p.tile1 * kKeys, s.len); ++key) {
          const uint32_t at = a.tables[(uint64_t)p.seq * a.table_width + key / a.cache.page_size];
          if (!view[h].sees(key) || at >= a.cache.pages) continue;
          const T* from = reinterpret_cast<const T*>(a.cache.v) +
                          (((uint64_t)at * a.cache.kv_heads + p.head) * a.cache.page_size +
                           key % a.cache.page_size) * kDim + c0;
#pragma unroll
          for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float v = (float)from[i * 8 + u];
              if (!(fabsf(v) < INFINITY)) y[i][u] += v;
            }
        }
      }
      if (p.partial >= 0) {
        const int r = r0 + 8 * h;
        float* rec = a.partial + (size_t)p.partial * partial_words<kRows, kDim>();
#pragma unroll
        for (int i = 0; i < kDim / 8; ++i)
          *reinterpret_cast<float2*>(rec + r * kDim + i * 8 + c0) = make_float2(y[i][0], y[i][1]);
        if (c0 == 0) {
          rec[kRows * kDim + r] = m[h] == -INFINITY ? m[h] : m[h] - F::kRaise;
          rec[kRows * kDim + kRows + r] = l[h];
        }
      } else {
        const float inv = l[h] == 0.f ? 0.f : __frcp_rn(l[h]);
        T* out = static_cast<T*>(a.out.data) + (uint64_t)(s.q0 + row[h] / a.group) * a.out.row_stride +
                 (uint64_t)(p.head * a.group + row[h] % a.group) * a.out.head_stride + c0;
#pragma unroll
        for (int i = 0; i < kDim / 8; ++i)
          *reinterpret_cast<uint32_t*>(out + i * 8) =
              Elements<T>::pair(__fmul_rn(y[i][0], inv), __fmul_rn(y[i][1], inv));
      }
    }
  }
  if (stop) ring.drain(used);
  __syncthreads();
  if (*abort_flag && tid == 0) mark_timeout();
}

template <class T, int kDim, int kTiles>
uint32_t launch(AttnArgs a, cudaStream_t s) {
  using C = Few<kDim, kTiles>;
  auto kernel = attention_few_kernel<T, kDim, kTiles>;
  static std::atomic<uint64_t> configured{0};
  if (attribute_needed(configured)) {
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::bytes(PB_MAX_SEQS)));
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    attribute_done(configured);
  }
  Maps maps{};
  uint32_t st = cache_maps<T>(a, kDim, C::kKeys, &maps);
  if (st) return st;
  const uint32_t grid = tree_ctas(C::kCtas);
  place_workspace(a, grid * kWarps, C::kRows, kDim);
  kernel<<<grid, kThreads, C::bytes(a.seqs), s>>>(a, maps);
  PB_CUDA(cudaGetLastError());
  return launch_combine<T, kDim, C::kRows>(a, grid * kWarps, s);
}

template <class T>
uint32_t by_size(const AttnArgs& a, uint32_t head_dim, uint32_t tiles, cudaStream_t s) {
  if (head_dim == 128) return launch<T, 128, 1>(a, s);
  return tiles == 1 ? launch<T, 64, 1>(a, s) : launch<T, 64, 2>(a, s);
}

}  // namespace

uint64_t few_tree_words(uint32_t head_dim, uint32_t tiles) {
  const int ctas = head_dim == 128 ? Few<128, 1>::kCtas : tiles == 1 ? Few<64, 1>::kCtas : Few<64, 2>::kCtas;
  return tree_words((uint64_t)tree_ctas(ctas) * kWarps, 16 * tiles, head_dim);
}

uint32_t few_timeouts(cudaStream_t s, uint32_t* count) { return add_timeouts(s, count); }

uint32_t few_tree(const AttnArgs& a, uint32_t type, uint32_t head_dim, uint32_t tiles, cudaStream_t s) {
  return type == PB_TYPE_F16 ? by_size<__half>(a, head_dim, tiles, s)
                             : by_size<__nv_bfloat16>(a, head_dim, tiles, s);
}

}  // namespace paged
}  // namespace pb
