// Tree attention of few rows per sequence and key head (16-bit types): single
// tokens and small drafts, where the keys and values are read once from memory and
// little is computed on them.
//
// At most 64 rows against a tile of 64 keys: four consumer warps, each with 16 rows
// (kTiles row groups) and its share of the tile's keys (4 / kTiles shares), run the
// online softmax of pb_attention_simt.cu on mma.sync m16n8k16 products, whose
// accumulators are the next product's operand as they stand; a fifth warp brings the
// tiles by TMA (128-byte swizzle) into a ring.  The legacy tensor path is the right
// one here: a tcgen05 tile has 128 rows, so that one token of seven heads would pay
// for 18 times its products, and its scores would pass through TMEM on the way.
// Bound by memory: the ring holds 64 KB at least per CTA, two CTAs per SM.
#include "pb_attention_launch.h"
#include "pb_attention_tma.cuh"

namespace pb {
namespace paged {
namespace {

constexpr int kConsumers = 4;
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kKeys = 64;
constexpr int kLeast = 2;

template <int kDim, int kTiles>
struct Few {
  static constexpr int kRows = 16 * kTiles;
  static constexpr int kShares = kConsumers / kTiles;   // of a tile's keys
  static constexpr int kShare = kKeys / kShares;        // keys of a warp
  static constexpr int kStages = kDim == 64 ? 5 : kShares > 1 ? 2 : 3;
  static constexpr int kHalves = kDim / 64;
  static constexpr int kBlock = kKeys * 128;
  static constexpr int kTile = kHalves * kBlock;        // K or V
  static constexpr int kJoinOff = kStages * 2 * kTile;  // shares joined: (kShares - 1) x 16 rows per row group
  static constexpr int kJoin = kShares > 1 ? (kShares - 1) * kRows * (kDim + 2) * 4 : 0;
  static constexpr int kBarOff = kJoinOff + kJoin;
  static constexpr int kPrefixOff = kBarOff + 2 * kStages * 8 + 16;
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
__global__ void __launch_bounds__(kThreads, 2)
attention_few_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Maps maps) {
  using C = Few<kDim, kTiles>;
  using F = Format<T>;
  constexpr int kRows = C::kRows, kStages = C::kStages, kHalves = C::kHalves, kShare = C::kShare;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  float* join = reinterpret_cast<float*>(smem + C::kJoinOff);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + kStages);
  volatile int* dirty = abort_flag + 1;  // the last piece with a value that was taken out
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + C::kPrefixOff);

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumers);
    }
    *abort_flag = 0;
    *dirty = 0;
    fence_barrier_init();
  }
  work_prefix<true, kRows, kKeys, kThreads>(a, prefix);  // ends with a barrier of the block
  const uint32_t total = prefix[a.seqs - 1];
  if (total == 0) return;
  const Share<kLeast> share(total, gridDim.x);
  if (blockIdx.x >= share.ctas) return;
  uint32_t next = share.start(blockIdx.x);
  const uint32_t end = share.start(blockIdx.x + 1);

  Sequence s;
  uint32_t rows;
  auto take = [&](Piece& p) { take_piece<true, kRows, kKeys>(a, prefix, next, end, p, s, rows); };

  if (warp == kConsumers) {
    const uint32_t leader = elect_one();
    int q = 0, brought = 0;
    bool stop = false;
    const uint32_t size = min(a.cache.page_size, (uint32_t)kKeys);  // keys of a box
    const uint32_t ring = smem_u32(smem);
    while (next < end && !stop) {
      Piece p;
      take(p);
      auto boxes = [&](uint32_t tile) { return min((uint32_t)kKeys / size, ceil_div(s.len - tile * kKeys, size)); };
      auto page_of = [&](uint32_t tile) {  // of box `lane` of a tile
        const uint32_t key = tile * kKeys + lane * size;
        return tile < p.tile1 && (uint32_t)lane < boxes(tile)
                   ? (int)a.tables[(uint64_t)p.seq * a.table_width + key / a.cache.page_size] : 0;
      };
      int page = page_of(p.tile0);
      for (uint32_t tile = p.tile0; tile < p.tile1; ++tile, ++q) {
        const int st = q % kStages, ahead = page_of(tile + 1);
        const uint32_t slot = tile * kKeys % a.cache.page_size, count = boxes(tile);
        if (!wait_soon(&empty[st], ((q / kStages) & 1) ^ 1, abort_flag)) { stop = true; break; }
        expect_tx(leader, &full[st], 2 * count * size * kHalves * 128);
        const uint32_t to = ring + st * 2 * C::kTile;
        for (uint32_t b = 0; b < count; ++b) {
          const int at = __shfl_sync(0xffffffffu, page, b);
#pragma unroll
          for (int c = 0; c < kHalves; ++c) {
            tma_4d(leader, to + c * C::kBlock + b * size * 128, &maps.k, c * 64, (int)slot, (int)p.head, at, &full[st]);
            tma_4d(leader, to + C::kTile + c * C::kBlock + b * size * 128, &maps.v, c * 64, (int)slot, (int)p.head, at,
                   &full[st]);
          }
        }
        brought = q + 1;
        page = ahead;
      }
    }
    if (*abort_flag)  // every copy lands before the CTA may exit
      for (int i = max(0, brought - kStages); i < brought; ++i)
        wait_drain(&full[i % kStages], (i / kStages) & 1, 50000000ull);
    __syncwarp();
  } else {
    const int group = warp % kTiles, part = warp / kTiles;  // rows 16 group.., keys kShare part.. of a tile
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;           // this thread's fragment row (and + 8) and column
    int q = 0, pieces = 0;
    bool stop = false;
    while (next < end && !stop) {
      Piece p;
      take(p);
      ++pieces;
      uint32_t row[2];
      RowView view[2];
      uint32_t qf[kDim / 16][4];  // Q as the first operand
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        row[h] = p.row_tile * kRows + group * 16 + r0 + 8 * h;
        const bool there = row[h] < rows;
        const uint32_t token = row[h] / a.group;
        view[h] = there ? row_view<true>(a, s, token) : RowView{0xffffffffu, 0ull};
        const T* src = static_cast<const T*>(a.q.data) + (uint64_t)(s.q0 + token) * a.q.row_stride +
                       (uint64_t)(p.head * a.group + row[h] % a.group) * a.q.head_stride + c0;
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k) {
          qf[k][h] = there ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
          qf[k][2 + h] = there ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
        }
      }
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      float o[kDim / 8][4];
#pragma unroll
      for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
      const uint32_t mask0 = s.context / kKeys;  // tiles from here on hold a key that some row does not see

      for (uint32_t tile = p.tile0; tile < p.tile1; ++tile, ++q) {
        const int st = q % kStages;
        if (!wait_soon(&full[st], (q / kStages) & 1, abort_flag)) { stop = true; break; }
        const uint32_t kt = smem_u32(smem) + st * 2 * C::kTile, vt = kt + C::kTile;
        const int k0 = part * kShare;  // this warp's keys in the tile
        float sc[kShare / 8][4];
#pragma unroll
        for (int j = 0; j < kShare / 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[j][i] = 0.f;
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k) {
#pragma unroll
          for (int j = 0; j < kShare / 16; ++j) {
            const int key = k0 + j * 16 + (lane >> 4) * 8 + (lane & 7), chunk = k * 2 + ((lane >> 3) & 1);
            uint32_t b[4];
            ldmatrix4(kt + chunk / 8 * C::kBlock + key * 128 + ((chunk % 8) ^ (key & 7)) * 16, b);
            mma16<T>(sc[2 * j], qf[k], b[0], b[1]);
            mma16<T>(sc[2 * j + 1], qf[k], b[2], b[3]);
          }
        }
        const bool masked = tile >= mask0;
        const uint32_t key0 = tile * kKeys + k0;
        if (masked) {
#pragma unroll
          for (int j = 0; j < kShare / 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!view[i / 2].sees(key0 + j * 8 + c0 + (i & 1))) sc[j][i] = -INFINITY;
        }
        float base[2];
        bool moved = false;
        float keep[2] = {1.f, 1.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = -INFINITY;
#pragma unroll
          for (int j = 0; j < kShare / 8; ++j) top = max_nan(top, sc[j][2 * h], sc[j][2 * h + 1]);
          top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1), -INFINITY);
          top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2), -INFINITY);
          top = __fmul_rn(top, a.scale_log2);
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
          for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = __fmul_rn(o[i][j], keep[j / 2]);
          l[0] = __fmul_rn(l[0], keep[0]);
          l[1] = __fmul_rn(l[1], keep[1]);
        }
        uint32_t pf[kShare / 16][4];  // P as the first operand
#pragma unroll
        for (int j = 0; j < kShare / 8; ++j) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = exp2_fast(__fmaf_rn(sc[j][i], a.scale_log2, base[i / 2]));
            l[i / 2] += w[i];
          }
          pf[j / 2][j % 2 * 2] = Elements<T>::pair(w[0], w[1]);
          pf[j / 2][j % 2 * 2 + 1] = Elements<T>::pair(w[2], w[3]);
        }
        if (masked) {
          // This warp's value rows: zero past the keys, and without what is not finite
          // (warps that share them find the same).
#pragma unroll
          for (int r = 0; r < kShare; r += 32) {
            const int key = k0 + r + lane;
            if (r + lane < kShare)
              if (clean_value_row<F, kDim, C::kBlock>(smem + st * 2 * C::kTile + C::kTile, key, tile * kKeys + key >= s.len))
                *dirty = pieces;
          }
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < kShare / 16; ++j) {
#pragma unroll
          for (int n = 0; n < kDim / 16; ++n) {
            const int key = k0 + j * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), chunk = n * 2 + (lane >> 4);
            uint32_t b[4];
            ldmatrix4_trans(vt + chunk / 8 * C::kBlock + key * 128 + ((chunk % 8) ^ (key & 7)) * 16, b);
            mma16<T>(o[2 * n], pf[j], b[0], b[1]);
            mma16<T>(o[2 * n + 1], pf[j], b[2], b[3]);
          }
        }
        if (masked) fence_async_smem();  // cleaned rows before the next copy over them
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }

      // The piece is done: the row sums, then the shares of a row group joined by its
      // first warp.  All consumers take the barriers, also on the way out.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      }
      if (C::kShares > 1) {
        auto record = [&](int share) { return join + (size_t)((share - 1) * kTiles + group) * 16 * (kDim + 2); };
        if (part > 0) {
          float* rec = record(part);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = r0 + 8 * h;
#pragma unroll
            for (int i = 0; i < kDim / 8; ++i)
              *reinterpret_cast<float2*>(rec + r * kDim + i * 8 + c0) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
            if (c0 == 0) {
              rec[16 * kDim + r] = m[h];
              rec[16 * kDim + 16 + r] = l[h];
            }
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (part == 0) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = r0 + 8 * h;
            float to = m[h];
#pragma unroll
            for (int i = 1; i < C::kShares; ++i) to = max_nan(to, record(i)[16 * kDim + r], -INFINITY);
            // a row that is not a number in one share is none in all
            auto weight = [&](float x) { return to == -INFINITY ? 0.f : exp2f(x - to); };
            const float w0 = weight(m[h]);
            l[h] = __fmul_rn(l[h], w0);
#pragma unroll
            for (int i = 0; i < kDim / 8; ++i) {
              o[i][2 * h] = __fmul_rn(o[i][2 * h], w0);
              o[i][2 * h + 1] = __fmul_rn(o[i][2 * h + 1], w0);
            }
#pragma unroll
            for (int i = 1; i < C::kShares; ++i) {
              const float* rec = record(i);
              const float w = weight(rec[16 * kDim + r]);
              l[h] = __fmaf_rn(w, rec[16 * kDim + 16 + r], l[h]);
#pragma unroll
              for (int n = 0; n < kDim / 8; ++n) {
                const float2 x = *reinterpret_cast<const float2*>(rec + r * kDim + n * 8 + c0);
                o[n][2 * h] = __fmaf_rn(w, x.x, o[n][2 * h]);
                o[n][2 * h + 1] = __fmaf_rn(w, x.y, o[n][2 * h + 1]);
              }
            }
            m[h] = to;
          }
        }
      } else {
        asm volatile("bar.sync 1, 128;" ::: "memory");  // every warp has looked at its values
      }
      const bool mend = *dirty == pieces;
      if (part == 0 && !stop) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (row[h] >= rows) continue;
          if (mend) {
            // A weight is positive: what is not finite passes through the sum as it is.
            for (uint32_t key = max(p.tile0, mask0) * kKeys; key < min(p.tile1 * kKeys, s.len); ++key) {
              const uint32_t page = a.tables[(uint64_t)p.seq * a.table_width + key / a.cache.page_size];
              if (!view[h].sees(key) || page >= a.cache.pages) continue;
              const T* from = reinterpret_cast<const T*>(a.cache.v) +
                              (((uint64_t)page * a.cache.kv_heads + p.head) * a.cache.page_size +
                               key % a.cache.page_size) * kDim + c0;
#pragma unroll
              for (int i = 0; i < kDim / 8; ++i) {
                const float x = (float)from[i * 8], y = (float)from[i * 8 + 1];
                if (!(fabsf(x) < INFINITY)) o[i][2 * h] += x;
                if (!(fabsf(y) < INFINITY)) o[i][2 * h + 1] += y;
              }
            }
          }
          const int r = group * 16 + r0 + 8 * h;
          if (p.partial >= 0) {
            float* rec = a.partial + (size_t)p.partial * partial_words<kRows, kDim>();
#pragma unroll
            for (int i = 0; i < kDim / 8; ++i)
              *reinterpret_cast<float2*>(rec + r * kDim + i * 8 + c0) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
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
                  Elements<T>::pair(__fmul_rn(o[i][2 * h], inv), __fmul_rn(o[i][2 * h + 1], inv));
          }
        }
      }
      // The joined shares have been read; and where one warp gave up, all end here.
      uint32_t gave_up;
      asm volatile(
          "{\n\t.reg .pred p, r;\n\t"
          "setp.ne.b32 p, %1, 0;\n\t"
          "barrier.cta.red.or.pred r, 1, 128, p;\n\t"
          "selp.u32 %0, 1, 0, r;\n\t}"
          : "=r"(gave_up)
          : "r"((uint32_t)stop)
          : "memory");
      if (gave_up) break;
    }
  }
  __syncthreads();
  if (*abort_flag && tid == 0) mark_timeout();
}

template <class T, int kDim, int kTiles>
uint32_t launch(const AttnArgs& a, cudaStream_t s) {
  using C = Few<kDim, kTiles>;
  auto kernel = attention_few_kernel<T, kDim, kTiles>;
  static std::atomic<uint64_t> configured{0};
  if (attribute_needed(configured)) {
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::bytes(PB_MAX_SEQS)));
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    attribute_done(configured);
  }
  Maps maps{};
  uint32_t st = cache_maps<T>(a, kDim, kKeys, &maps);
  if (st) return st;
  const uint32_t grid = tree_ctas(2);
  kernel<<<grid, kThreads, C::bytes(a.seqs), s>>>(a, maps);
  PB_CUDA(cudaGetLastError());
  return launch_combine<T, kDim, C::kRows, kKeys, kLeast>(a, grid, s);
}

template <class T>
uint32_t by_size(const AttnArgs& a, uint32_t head_dim, uint32_t tiles, cudaStream_t s) {
  if (head_dim == 64) return tiles == 1 ? launch<T, 64, 1>(a, s) : launch<T, 64, 2>(a, s);
  return tiles == 1 ? launch<T, 128, 1>(a, s) : launch<T, 128, 2>(a, s);
}

}  // namespace

uint64_t few_tree_words(uint32_t head_dim, uint32_t tiles) {
  return (uint64_t)tree_ctas(2) * 2 * 16 * tiles * (head_dim + 2);
}

uint32_t few_status() { return take_status(); }

uint32_t few_tree(const AttnArgs& a, uint32_t type, uint32_t head_dim, uint32_t tiles, cudaStream_t s) {
  return type == PB_TYPE_F16 ? by_size<__half>(a, head_dim, tiles, s)
                             : by_size<__nv_bfloat16>(a, head_dim, tiles, s);
}

}  // namespace paged
}  // namespace pb
