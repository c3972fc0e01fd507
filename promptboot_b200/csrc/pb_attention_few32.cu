// Tree attention of few rows per sequence and key head in binary32 (products and
// sums too): the counterpart of pb_attention_few.cu on the CUDA cores.
//
// Each warp walks a run of tiles through a ring of its own (128-byte swizzle).  Scores:
// a lane has a key, or half of one, and all rows, whose queries it reads from shared
// memory, the same word for every lane.  Weights go through shared memory; values: a
// lane has kDim / 32 elements and all rows.  The running maximum moves only where a
// score passes it by more than kSlack, so that it takes the warp's shuffles seldom.
//
// Bound by the latency of a warp's chain through a tile, with two or three warps to a
// scheduler (a third of its issue slots): 69 us for 256 single tokens over 512 to 1024
// positions, 14 heads of 64 to 2 (2.95 TB/s), 210 us for 16 over 6000, 32 heads of 128
// to 8 (3.5 TB/s).  The first took 138 us on row tiles of 16 of pb_attention_simt.cu.
#include "pb_attention_launch.h"
#include "pb_attention_tma.cuh"

namespace pb {
namespace paged {
namespace {

constexpr int kStages = 2;

template <int kDim, int kRows>
struct Few32 {
  // Ten warps with tiles of 8 KB of keys and values, or five with tiles of 16: ten are
  // faster where their sums leave the registers (64 x 8: 69 against 77 us for 256 single
  // tokens, 2.95 TB/s), five else (128 x 16: 209 against 233 us for 64 x 4 nodes).
  static constexpr bool kMany = kDim == 64 && kRows == 8;
  static constexpr int kWarps = kMany ? 10 : 5;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kLeast = kMany ? 4 : 2;         // tiles of a run
  static constexpr int kSplit = kMany ? 2 : kDim / 64; // lanes of a key
  static constexpr int kKeys = 32 / kSplit;
  static constexpr int kBlocks = kDim / 32;            // 128-byte column blocks of a row
  static constexpr int kBlock = kKeys * 128;
  static constexpr int kTile = kBlocks * kBlock;       // K or V
  static constexpr int kQOff = kWarps * kStages * 2 * kTile;
  static constexpr int kQ = kRows * kDim * 4;
  static constexpr int kPOff = kQOff + kWarps * kQ;
  static constexpr int kP = kKeys * kRows * 4;
  static constexpr int kBarOff = kPOff + kWarps * kP;
  static constexpr int kPrefixOff = kBarOff + kWarps * kStages * 8 + 16;
  static size_t bytes(uint32_t seqs) { return 1024 + kPrefixOff + (size_t)seqs * 4; }
};

template <int kDim, int kRows>
__global__ void __launch_bounds__(Few32<kDim, kRows>::kThreads, 1)
attention_few32_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Maps maps) {
  using C = Few32<kDim, kRows>;
  constexpr int kKeys = C::kKeys, kSplit = C::kSplit, kWarps = C::kWarps, kE = kDim / 32;  // elements of a lane
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kWarps * kStages);
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + C::kPrefixOff);

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  float* qs = reinterpret_cast<float*>(smem + C::kQOff + warp * C::kQ);
  float* ps = reinterpret_cast<float*>(smem + C::kPOff + warp * C::kP);
  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(&bars[i], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  work_prefix<true, kRows, kKeys, C::kThreads>(a, prefix);  // ends with a barrier of the block
  const uint32_t total = prefix[a.seqs - 1];
  const Share<C::kLeast> share(total, gridDim.x * kWarps);
  const uint32_t run = blockIdx.x * kWarps + warp;
  uint32_t next = run < share.runs ? share.start(run) : total;
  const uint32_t end = run < share.runs ? share.start(run + 1) : total;
  TileRing<float, kRows, kKeys, C::kBlocks, kStages> ring(a, maps, prefix, bars + warp * kStages,
                                                         smem + warp * kStages * 2 * C::kTile, next, end);
  if (lane == 0) note_join<kRows, kKeys>(a, prefix, share, run);

  const int key = lane / kSplit, part = lane % kSplit;  // of the scores
  const int d0 = lane * kE;                             // of the values
  Sequence s;
  uint32_t rows;
  int used = 0;  // tiles
  bool stop = false;
  while (next < end && !stop) {
    Piece p;
    take_piece<true, kRows, kKeys>(a, prefix, run, next, end, p, s, rows);
    const uint32_t first = p.row_tile * kRows;
    __syncwarp();
    for (int i = lane; i < kRows * (kDim / 4); i += 32) {
      const int r = i / (kDim / 4), c = i % (kDim / 4) * 4;
      const uint32_t row = first + r;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows)
        x = *reinterpret_cast<const float4*>(
            static_cast<const float*>(a.q.data) + (uint64_t)(s.q0 + row / a.group) * a.q.row_stride +
            (uint64_t)(p.head * a.group + row % a.group) * a.q.head_stride + c);
      *reinterpret_cast<float4*>(qs + r * kDim + c) = x;
    }
    __syncwarp();
    float m[kRows], l[kRows], o[kRows][kE];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int e = 0; e < kE; ++e) o[r][e] = 0.f;
    }
    const uint32_t mask0 = s.context / kKeys;  // tiles from here on hold a key that some row does not see

    for (uint32_t tile = p.tile0; tile < p.tile1; ++tile) {
      if (!wait_soon(&ring.full[used % kStages], (used / kStages) & 1, abort_flag)) { stop = true; break; }
      const uint8_t* kt = ring.keys(used++);
      const uint8_t* vt = kt + C::kTile;
      float x[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) x[r] = 0.f;
#pragma unroll 4
      for (int i = 0; i < C::kBlocks / kSplit * 8; ++i) {
        // the parts of a key take their words in other orders: their banks differ
        const int chunk = i % 8 ^ (part * (8 / kSplit)), block = part * (C::kBlocks / kSplit) + i / 8;
        const float4 k4 = *reinterpret_cast<const float4*>(kt + block * C::kBlock + key * 128 + ((chunk ^ (key & 7)) * 16));
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 q4 = *reinterpret_cast<const float4*>(qs + r * kDim + block * 32 + chunk * 4);
          x[r] = __fmaf_rn(q4.x, k4.x, x[r]);
          x[r] = __fmaf_rn(q4.y, k4.y, x[r]);
          x[r] = __fmaf_rn(q4.z, k4.z, x[r]);
          x[r] = __fmaf_rn(q4.w, k4.w, x[r]);
        }
      }
      const bool masked = tile >= mask0;
      const uint32_t key0 = tile * kKeys;
      bool over = false;
      uint32_t seen = 0xffffffffu;  // rows that see this lane's key
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int d = 1; d < kSplit; d <<= 1) x[r] += __shfl_xor_sync(0xffffffffu, x[r], d);
        x[r] = __fmul_rn(x[r], a.scale_log2);
        if (masked) {
          const uint32_t row = first + r;
          // Rows past the last see nothing here: a slot without a key would else decide
          // whether the maxima move, and with that how the other rows round.
          if (row >= rows || !row_view<true>(a, s, row / a.group).sees(key0 + key)) {
            seen &= ~(1u << r);
            x[r] = -INFINITY;
          }
        }
        over |= !(x[r] <= m[r] + Format<float>::kSlack);
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          float top = x[r];
#pragma unroll
          for (int d = 16; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d), -INFINITY);
          if (!(top < INFINITY)) {
            m[r] = NAN;  // a score that is not a number or +inf: so is the row
          } else if (m[r] == -INFINITY) {
            m[r] = top;  // nothing has been added yet
          } else if (top > m[r]) {
            const float keep = exp2f(m[r] - top);
            m[r] = top;
            l[r] = __fmul_rn(l[r], keep);
#pragma unroll
            for (int e = 0; e < kE; ++e) o[r][e] = __fmul_rn(o[r][e], keep);
          }
        }
      }
      // A key that a row does not see gets the weight -0, by which its value is left out
      // whatever it holds.
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float w = exp2_fast(x[r] - (m[r] == -INFINITY ? 0.f : m[r]));
        if (part == 0) l[r] += w;
        x[r] = (seen >> r) & 1 ? w : -0.f;
      }
      if (part == 0) {
#pragma unroll
        for (int r = 0; r < kRows; r += 4)
          *reinterpret_cast<float4*>(ps + key * kRows + r) = make_float4(x[r], x[r + 1], x[r + 2], x[r + 3]);
      }
      __syncwarp();
      auto add_values = [&](auto checked) {
#pragma unroll 4
        for (int j = 0; j < kKeys; ++j) {
          const uint8_t* at = vt + d0 / 32 * C::kBlock + j * 128 + ((d0 % 32 / 4) ^ (j & 7)) * 16 + d0 % 4 * 4;
          float v[kE];
          if (kE == 2) {
            const float2 t = *reinterpret_cast<const float2*>(at);
            v[0] = t.x;
            v[1] = t.y;
          } else {
            const float4 t = *reinterpret_cast<const float4*>(at);
            v[0] = t.x;
            v[1] = t.y;
            v[kE - 2] = t.z;
            v[kE - 1] = t.w;
          }
#pragma unroll
          for (int r = 0; r < kRows; r += 4) {
            const float4 w4 = *reinterpret_cast<const float4*>(ps + j * kRows + r);
            const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              if (decltype(checked)::value && __float_as_uint(w[u]) == 0x80000000u) continue;
#pragma unroll
              for (int e = 0; e < kE; ++e) o[r + u][e] = __fmaf_rn(w[u], v[e], o[r + u][e]);
            }
          }
        }
      };
      if (masked) add_values(std::true_type{});
      else add_values(std::false_type{});
      __syncwarp();
      ring.send();
    }
    if (stop) break;

    // The piece is done: O / l, or O with its maximum and sum.
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int d = 16; d; d >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
      const uint32_t row = first + r;
      if (row >= rows) continue;
      float* to;
      float by = 1.f;
      if (p.partial >= 0) {
        float* rec = a.partial + (size_t)p.partial * partial_words<kRows, kDim>();
        to = rec + r * kDim + d0;
        if (lane == 0) {
          rec[kRows * kDim + r] = m[r];
          rec[kRows * kDim + kRows + r] = l[r];
        }
      } else {
        by = l[r] == 0.f ? 0.f : 1.f / l[r];
        to = static_cast<float*>(a.out.data) + (uint64_t)(s.q0 + row / a.group) * a.out.row_stride +
             (uint64_t)(p.head * a.group + row % a.group) * a.out.head_stride + d0;
      }
      if (kE == 2)
        *reinterpret_cast<float2*>(to) = make_float2(o[r][0] * by, o[r][1] * by);
      else
        *reinterpret_cast<float4*>(to) = make_float4(o[r][0] * by, o[r][1] * by, o[r][kE - 2] * by, o[r][kE - 1] * by);
    }
  }
  if (stop) ring.drain(used);
  __syncthreads();
  if (*abort_flag && tid == 0) mark_timeout();
}

template <int kDim, int kRows>
uint32_t launch(AttnArgs a, cudaStream_t s) {
  using C = Few32<kDim, kRows>;
  auto kernel = attention_few32_kernel<kDim, kRows>;
  static std::atomic<uint64_t> configured{0};
  if (attribute_needed(configured)) {
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::bytes(PB_MAX_SEQS)));
    attribute_done(configured);
  }
  Maps maps{};
  uint32_t st = cache_maps<float>(a, kDim, C::kKeys, &maps);
  if (st) return st;
  const uint32_t grid = tree_ctas(1);
  place_workspace(a, grid * C::kWarps, kRows, kDim);
  kernel<<<grid, C::kThreads, C::bytes(a.seqs), s>>>(a, maps);
  PB_CUDA(cudaGetLastError());
  return launch_combine<float, kDim, kRows>(a, grid * C::kWarps, s);
}

}  // namespace

uint64_t few32_tree_words(uint32_t head_dim, uint32_t tile_rows) {
  const uint32_t warps = head_dim == 64 && tile_rows == 8 ? Few32<64, 8>::kWarps : Few32<64, 16>::kWarps;
  return tree_words((uint64_t)tree_ctas(1) * warps, tile_rows, head_dim);
}

uint32_t few32_tree(const AttnArgs& a, uint32_t head_dim, uint32_t tile_rows, cudaStream_t s) {
  if (head_dim == 64) return tile_rows == 8 ? launch<64, 8>(a, s) : launch<64, 16>(a, s);
  return tile_rows == 8 ? launch<128, 8>(a, s) : launch<128, 16>(a, s);
}

uint32_t few32_timeouts(cudaStream_t s, uint32_t* count) { return add_timeouts(s, count); }

}  // namespace paged
}  // namespace pb
