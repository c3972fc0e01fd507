// Paged serving attention on the 5th-generation tensor cores (tcgen05, kind::f16)
// for binary16 and bfloat16: prompts, and trees with many rows per sequence.
//
// A CTA walks the keys of one row tile (128 rows) in tiles of kKeys, with the
// online softmax of pb_attention_simt.cu in binary32:
//   S = Q K^T (both from shared memory, S in TMEM),  P = 2^(S c - m) rounded to
//   the type of V (into TMEM),  O += P V (P from TMEM, V from shared memory).
// The weights' sum adds the unrounded weights, so P's rounding is one more half
// step of the type per weight and averages out over the keys.
//
// A CTA has kGroups row tiles, which share the K and V tiles that pass by.  Each has
// four softmax warps, one row per thread (TMEM lane = row), and a warp that issues its
// MMAs; one more warp brings K and V tiles by TMA (128-byte swizzle) into rings of
// kStages.  S, P and O have TMEM columns of their own: the scores of the next tile go
// out as soon as those of this one are in registers, under its exponentials.
//
// Bound by the softmax warps: per key and row an exponential (16 a cycle and SM) and
// some five other instructions, in dependent chains that one or two warps per
// scheduler leave half idle (50% issue).  So three row tiles at heads of 64 (480 of
// 512 TMEM columns, one CTA per SM, three softmax warps per scheduler) where a sequence
// fills them, else one row tile and two CTAs per SM.
//
// The running maximum is the one in use until a row's true maximum passes it by
// 2^kSlack: O is rescaled (through registers) only then, seldom after the first
// tiles.  Weights may then reach 2^kSlack; binary16 weights are also raised by
// 2^kRaise, so that those far below the maximum keep their bits.
//
// Masked tiles (a key that some row of the tile does not see): scores are replaced
// by -inf; value rows past the keys are zeroed in shared memory; values that are
// not finite are taken out there, and added to the rows that see them at the end.
#include "pb_attention_launch.h"
#include "pb_attention_tma.cuh"

namespace pb {
namespace paged {

namespace {

constexpr int kRowTile = 128;  // rows of one MMA
constexpr int kKeys = 64;
constexpr int kLeast = 2;

template <int kDim, int kGroups>
struct Tc {
  static constexpr int kRows = kGroups * kRowTile;
  static constexpr int kThreads = 32 * (5 * kGroups + 1);
  static constexpr int kCtas = kGroups == 1 ? 2 : 1;  // per SM
  static constexpr int kStages = kGroups > 1 ? 5 : kDim == 64 ? 4 : 2;
  static constexpr int kHalves = kDim / 64;            // 128-byte column blocks of a row
  static constexpr int kQBlock = kRowTile * 128;
  static constexpr int kQ = kHalves * kQBlock;         // Q of one row tile
  static constexpr int kBlock = kKeys * 128;           // one column block of a K or V tile
  static constexpr int kTile = kHalves * kBlock;
  static constexpr int kKOff = kGroups * kQ;
  static constexpr int kVOff = kKOff + kStages * kTile;
  static constexpr int kBarOff = kVOff + kStages * kTile;
  static constexpr int kBars = 4 * kStages + 6 * kGroups;
  static constexpr int kPrefixOff = kBarOff + kBars * 8 + 16;
  static constexpr int kPCol = kKeys, kOCol = kKeys + kKeys / 2, kGroupCols = kOCol + kDim;
  static constexpr int kCols = kCtas == 2 ? 256 : 512;
  static_assert(kGroups * kGroupCols <= kCols, "TMEM columns");
  static size_t bytes(uint32_t seqs) { return 1024 + kPrefixOff + (size_t)seqs * 4; }
};

__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit_to(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// Waits for this thread's TMEM loads; the registers pass through, so that nothing
// that uses them moves up.
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[N]) {
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Shared-memory matrix descriptor, 128-byte swizzle (8 rows of 128 bytes repeat):
// stride 1024 bytes between 8-row groups.  `lead`: bytes between 64-element column
// blocks of an N-major operand (V); unused by K-major ones (Q, K).
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float x0, x1;
  unpk(x, x0, x1);
  return pk(exp2_fast(x0), exp2_fast(x1));
}
// The same without the exponential unit: x less its nearest whole number n (Cody and
// Waite's reduction; n comes out of the low bits of x + 1.5 * 2^23) through a
// polynomial of least relative error on [-1/2, 1/2], 7.5e-5 of degree 3 and 2.6e-6
// of degree 4, times 2^n by an addition to the exponent.  x from -126 (below: 2^-126
// at most) to 127.
template <int kDegree>
__device__ __forceinline__ uint64_t exp2_poly(uint64_t x) {
  float x0, x1;
  unpk(x, x0, x1);
  x = pk(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t t = add2(x, pk(12582912.f, 12582912.f));
  const uint64_t f = fma2(add2(t, pk(-12582912.f, -12582912.f)), pk(-1.f, -1.f), x);
  auto both = [](float c) { return pk(c, c); };
  uint64_t y;
  if (kDegree == 3) {
    y = fma2(both(0.055171669f), f, both(0.242611125f));
    y = fma2(y, f, both(0.693260968f));
    y = fma2(y, f, both(0.999928057f));
  } else {
    y = fma2(both(0.0095701022f), f, both(0.0559178628f));
    y = fma2(y, f, both(0.240247443f));
    y = fma2(y, f, both(0.693121791f));
    y = fma2(y, f, both(0.999999285f));
  }
  float y0, y1, t0, t1;
  unpk(y, y0, y1);
  unpk(t, t0, t1);
  return pk_u(__float_as_uint(y0) + (__float_as_uint(t0) << 23), __float_as_uint(y1) + (__float_as_uint(t1) << 23));
}
// Which of the 32 keys from `key` on a row sees.
__device__ __forceinline__ uint32_t seen32(const RowView& r, uint32_t key) {
  const uint32_t below = r.all > key ? r.all - key : 0;
  if (below >= 32) return 0xffffffffu;
  uint32_t m = (1u << below) - 1u;
  if (key >= r.all) {
    const uint32_t at = key - r.all;
    if (at < 64) m |= (uint32_t)(r.bits >> at);
  } else {
    m |= (uint32_t)(r.bits << below);
  }
  return m;
}

template <class T, int kDim, int kGroups, bool kTree>
__global__ void __launch_bounds__(Tc<kDim, kGroups>::kThreads, Tc<kDim, kGroups>::kCtas)
attention_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Maps maps) {
  using C = Tc<kDim, kGroups>;
  using F = Format<T>;
  constexpr int kRows = C::kRows, kStages = C::kStages, kHalves = C::kHalves;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* groups = v_empty + kStages;  // six per row tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(groups + 6 * kGroups);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* dirty = abort_flag + 1;  // the last piece with a value that was taken out
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + C::kPrefixOff);

  if (kTree) pdl_trigger();
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  work_prefix<kTree, kRows, kKeys, C::kThreads>(a, prefix);
  const uint32_t total = prefix[a.seqs - 1];
  uint32_t next, end;
  if (kTree) {
    if (total == 0) return;
    const Share<kLeast> share(total, gridDim.x);
    if (blockIdx.x >= share.ctas) return;
    next = share.start(blockIdx.x);
    end = share.start(blockIdx.x + 1);
  } else {
    if (blockIdx.x >= total) return;
    next = blockIdx.x;
    end = next + 1;
  }

  if (warp == 0) tmem_alloc(tmem_slot, C::kCols);
  if (tid == 32) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], kGroups);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], kGroups);
    }
    for (int g = 0; g < kGroups; ++g) {
      mbar_init(&groups[6 * g], 4);
      mbar_init(&groups[6 * g + 1], 1);
      mbar_init(&groups[6 * g + 2], 4);
      mbar_init(&groups[6 * g + 3], 4);
      mbar_init(&groups[6 * g + 4], 1);
      mbar_init(&groups[6 * g + 5], 1);
    }
    *abort_flag = 0;
    *dirty = 0;
    fence_barrier_init();
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();

  // The row tile of a softmax or MMA warp: its TMEM columns and barriers.
  const int group = warp < 4 * kGroups ? warp >> 2 : min(warp - 4 * kGroups, kGroups - 1);
  const uint32_t tmem = *tmem_slot + group * C::kGroupCols;
  uint64_t* q_full = groups + 6 * group;  // Q is in shared memory
  uint64_t* s_full = q_full + 1;          // S holds a tile's scores
  uint64_t* s_free = q_full + 2;          // they are in registers
  uint64_t* p_full = q_full + 3;          // P holds its weights
  uint64_t* o_full = q_full + 4;          // O holds its products, P is free
  uint64_t* drained = q_full + 5;         // on the way out: every issued MMA has ended

  // The CTA's pieces, decoded alike by every role; and the last key tile that some row
  // of this row tile sees.
  Sequence s;
  uint32_t rows;
  auto take = [&](Piece& p) { take_piece<kTree, kRows, kKeys>(a, prefix, next, end, p, s, rows); };
  auto first_row = [&](const Piece& p) { return p.row_tile * kRows + group * kRowTile; };
  auto tiles_of = [&](const Piece& p) {
    const uint32_t r0 = first_row(p);
    if (r0 >= rows) return p.tile0;
    if (kTree) return p.tile1;
    const uint32_t last = min(rows, r0 + kRowTile) - 1;
    return min(p.tile1, ceil_div(row_view<false>(a, s, last / a.group).all, kKeys));
  };

  if (warp == 5 * kGroups) {
    const uint32_t leader = elect_one();
    const uint32_t size = kTree ? min(a.cache.page_size, (uint32_t)kKeys) : kKeys;  // keys of a box
    const uint32_t ka = smem_u32(smem) + C::kKOff, va = smem_u32(smem) + C::kVOff;
    int q = 0, k_brought = 0, v_brought = 0;  // tiles so far
    bool stop = false;
    while (next < end && !stop) {
      Piece p;
      take(p);
      auto boxes = [&](uint32_t tile) { return min((uint32_t)kKeys / size, ceil_div(s.len - tile * kKeys, size)); };
      auto page_of = [&](uint32_t tile) {  // of box `lane` of a tile
        const uint32_t key = tile * kKeys + lane * size;
        return kTree && tile < p.tile1 && (uint32_t)lane < boxes(tile)
                   ? (int)a.tables[(uint64_t)p.seq * a.table_width + key / a.cache.page_size] : 0;
      };
      int page = page_of(p.tile0);
      for (uint32_t tile = p.tile0; tile < p.tile1; ++tile, ++q) {
        const int st = q % kStages, ahead = page_of(tile + 1);
        const uint32_t key = tile * kKeys, count = boxes(tile);
        auto bring = [&](uint32_t to, const CUtensorMap* map, uint32_t step, uint64_t* full) {
          expect_tx(leader, full, count * size * kHalves * 128);
          for (uint32_t b = 0; b < count; ++b) {
            const int at = kTree ? __shfl_sync(0xffffffffu, page, b) : 0;
#pragma unroll
            for (int c = 0; c < kHalves; ++c) {
              if (kTree)
                tma_4d(leader, to + c * C::kBlock + b * size * 128, map, c * 64, (int)(key % a.cache.page_size),
                       (int)p.head, at, full);
              else
                tma_3d(leader, to + c * C::kBlock, map, c * 64, (int)(s.kv0 + key), (int)(p.head * step), full);
            }
          }
        };
        if (!wait_soon(&k_empty[st], ((q / kStages) & 1) ^ 1, abort_flag)) { stop = true; break; }
        bring(ka + st * C::kTile, &maps.k, maps.k_step, &k_full[st]);
        k_brought = q + 1;
        if (!wait_soon(&v_empty[st], ((q / kStages) & 1) ^ 1, abort_flag)) { stop = true; break; }
        bring(va + st * C::kTile, &maps.v, maps.v_step, &v_full[st]);
        v_brought = q + 1;
        page = ahead;
      }
    }
    if (*abort_flag) {  // every copy lands before the CTA may exit
      for (int i = max(0, k_brought - kStages); i < k_brought; ++i)
        wait_drain(&k_full[i % kStages], (i / kStages) & 1, 50000000ull);
      for (int i = max(0, v_brought - kStages); i < v_brought; ++i)
        wait_drain(&v_full[i % kStages], (i / kStages) & 1, 50000000ull);
    }
    __syncwarp();
  } else if (warp >= 4 * kGroups) {
    const uint32_t leader = elect_one();
    constexpr uint32_t kBase = (1u << 4) | (F::kCode << 7) | (F::kCode << 10) | ((uint32_t)(kRowTile >> 4) << 24);
    constexpr uint32_t kQk = kBase | ((uint32_t)(kKeys >> 3) << 17);
    constexpr uint32_t kPv = kBase | ((uint32_t)(kDim >> 3) << 17) | (1u << 16);  // V is N-major
    const uint32_t qa = smem_u32(smem) + group * C::kQ;
    const uint32_t ka = smem_u32(smem) + C::kKOff, va = smem_u32(smem) + C::kVOff;
    int q = 0, t = 0, walked = 0;  // tiles that passed by; this row tile's; its pieces with tiles
    bool stop = false;
    while (next < end && !stop) {
      Piece p;
      take(p);
      const int n = (int)(p.tile1 - p.tile0), mine = (int)(tiles_of(p) - p.tile0);
      auto scores = [&](int i) {  // S = Q K^T of tile i
        const int st = (q + i) % kStages;
        if (!wait_soon(&k_full[st], ((q + i) / kStages) & 1, abort_flag)) return false;
        tc_after_sync();
#pragma unroll
        for (int j = 0; j < kDim / 16; ++j)
          mma_ss(leader, tmem, desc128(qa + j / 4 * C::kQBlock + j % 4 * 32, 16),
                 desc128(ka + st * C::kTile + j / 4 * C::kBlock + j % 4 * 32, 16), kQk, j > 0);
        commit_to(leader, s_full);
        commit_to(leader, &k_empty[st]);
        return true;
      };
      if (mine > 0) {
        if (!wait_soon(q_full, walked & 1, abort_flag) || !scores(0)) break;
        ++walked;
      }
      for (int i = 0; i < mine; ++i, ++t) {
        const int st = (q + i) % kStages;
        if ((i + 1 < mine && (!wait_soon(s_free, t & 1, abort_flag) || !scores(i + 1))) ||
            !wait_soon(p_full, t & 1, abort_flag) ||
            !wait_soon(&v_full[st], ((q + i) / kStages) & 1, abort_flag)) {
          stop = true;
          break;
        }
        tc_after_sync();
#pragma unroll
        for (int j = 0; j < kKeys / 16; ++j)
          mma_ts(leader, tmem + C::kOCol, tmem + C::kPCol + j * 8, desc128(va + st * C::kTile + j * 2048, C::kBlock),
                 kPv, i > 0 || j > 0);
        commit_to(leader, o_full);
        commit_to(leader, &v_empty[st]);
      }
      for (int i = max(0, mine); i < n && !stop; ++i) {  // tiles for the other row tiles alone
        const int st = (q + i) % kStages;
        stop = !wait_soon(&k_full[st], ((q + i) / kStages) & 1, abort_flag) ||
               !wait_soon(&v_full[st], ((q + i) / kStages) & 1, abort_flag);
        if (!stop && lane == 0) {
          mbar_arrive(&k_empty[st]);
          mbar_arrive(&v_empty[st]);
        }
        __syncwarp();
      }
      q += n;
    }
    if (*abort_flag) {
      commit_to(leader, drained);
      wait_drain(drained, 0, 50000000ull);
    }
    __syncwarp();
  } else {
    const int me = tid & (kRowTile - 1);
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);  // this warp's lanes
    uint8_t* q_tile = smem + group * C::kQ;
    int q = 0, t = 0, pieces = 0;  // tiles that passed by; this row tile's; pieces
    bool stop = false;
    while (next < end && !stop) {
      Piece p;
      take(p);
      ++pieces;
      const uint32_t row = first_row(p) + me, token = row / a.group;
      const uint32_t head = p.head * a.group + row % a.group;
      const bool there = row < rows;
      // Rows past the last see everything: zeros times finite or other keys, never stored.
      const RowView view = there ? row_view<kTree>(a, s, token) : RowView{0xffffffffu, 0ull};
      float m = -INFINITY;      // the maximum in use, in powers of two
      uint64_t l2[2] = {0, 0};  // the sum of weights, in four parts
      // Tiles from here on hold a key that some row of this row tile, of the CTA does not see.
      auto blind = [&](uint32_t r) { return (kTree ? s.context : row_view<false>(a, s, r / a.group).all) / kKeys; };
      const uint32_t tile1 = tiles_of(p), mask0 = p.tile0 < tile1 ? blind(first_row(p)) : 0;
      if (p.tile0 < tile1) {
        const T* src = static_cast<const T*>(a.q.data) + (uint64_t)(s.q0 + token) * a.q.row_stride +
                       (uint64_t)head * a.q.head_stride;
#pragma unroll
        for (int c = 0; c < kDim / 8; ++c) {
          const uint4 w = there ? reinterpret_cast<const uint4*>(src)[c] : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(q_tile + c / 8 * C::kQBlock + me * 128 + ((c % 8) ^ (me & 7)) * 16) = w;
        }
        fence_async_smem();
        tc_before_sync();  // the piece before has been read from TMEM
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      for (uint32_t tile = p.tile0; tile < tile1; ++tile, ++t) {
        const uint32_t key0 = tile * kKeys;
        const bool masked = tile >= mask0;
        if (!wait_soon(s_full, t & 1, abort_flag)) { stop = true; break; }
        tc_after_sync();
        uint32_t v[2][32];
        tmem_ld32(tl, v[0]);
        tmem_ld32(tl + 32, v[1]);
        tmem_wait(v[0]);
        tmem_wait(v[1]);
        tc_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        if (masked) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t seen = seen32(view, key0 + 32 * c);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[c][i] = (seen >> i) & 1 ? v[c][i] : 0xff800000u;  // -inf
          }
        }
        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            top4[u] = max_nan(top4[u], __uint_as_float(v[i / 32][i % 32 + 2 * u]),
                              __uint_as_float(v[i / 32][i % 32 + 2 * u + 1]));
        const float top =
            __fmul_rn(max_nan(max_nan(top4[0], top4[1], top4[2]), top4[3], top4[3]), a.scale_log2);
        // P and O are free when the products before are done.
        if (t > 0 && !wait_soon(o_full, (t - 1) & 1, abort_flag)) { stop = true; break; }
        tc_after_sync();
        float keep = 1.f;
        if (!(top < INFINITY)) {
          m = NAN;  // a score that is not a number or +inf: so is the row
        } else if (m == -INFINITY) {
          m = top;  // O holds zeros at most
        } else if (top > m + F::kSlack) {
          keep = exp2_fast(m - top);
          m = top;
        }
        if (__any_sync(0xffffffffu, keep != 1.f)) {  // never in a piece's first tile
          uint32_t o[16];
#pragma unroll
          for (int c = 0; c < kDim; c += 16) {
            tmem_ld16(tl + C::kOCol + c, o);
            tmem_wait(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__fmul_rn(__uint_as_float(o[i]), keep));
            tmem_st16(tl + C::kOCol + c, o);
          }
          l2[0] = mul2(l2[0], pk(keep, keep));
          l2[1] = mul2(l2[1], pk(keep, keep));
        }
        const float base = F::kRaise - (m == -INFINITY ? 0.f : m);
        const uint64_t scale2 = pk(a.scale_log2, a.scale_log2), base2 = pk(base, base);
        // One exponential in four through the polynomial; all through the unit where keys
        // are masked, whose weight has to be zero.
        auto weigh = [&](auto mixed) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              uint64_t y = fma2(pk_u(v[c][i], v[c][i + 1]), scale2, base2);
              y = decltype(mixed)::value && i % 8 == 6 ? exp2_poly<F::kDegree>(y) : exp2_pair(y);
              l2[i / 2 & 1] = add2(l2[i / 2 & 1], y);
              float y0, y1;
              unpk(y, y0, y1);
              w[i / 2] = Elements<T>::pair(y0, y1);
            }
            tmem_st16(tl + C::kPCol + 16 * c, w);
          }
        };
        if (masked) weigh(std::false_type{});
        else weigh(std::true_type{});
        if (masked) {
          // Value rows of this tile, one per thread: zero past the keys, and without
          // what is not finite (row tiles that share them find the same).
          const int at = q + (int)(tile - p.tile0);
          if (!wait_soon(&v_full[at % kStages], (at / kStages) & 1, abort_flag)) { stop = true; break; }
          if (me < kKeys)
            clean_value_row<F, kDim, C::kBlock>(smem + C::kVOff + at % kStages * C::kTile, me, key0 + me >= s.len,
                                                dirty, pieces);
          fence_async_smem();
        }
        tmem_wait_st();
        tc_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      q += (int)(p.tile1 - p.tile0);
      if (stop) break;

      // The piece is done: O / l, or O with its maximum and sum.
      if (p.tile0 < tile1) {
        if (!wait_soon(o_full, (t - 1) & 1, abort_flag)) break;
        tc_after_sync();
      }
      float part[4];
      unpk(l2[0], part[0], part[1]);
      unpk(l2[1], part[2], part[3]);
      const float l = (part[0] + part[1]) + (part[2] + part[3]);
      const float inv = l == 0.f ? 0.f : __frcp_rn(l);
      T* out = static_cast<T*>(a.out.data) + (uint64_t)(s.q0 + token) * a.out.row_stride +
               (uint64_t)head * a.out.head_stride;
      const int in_tile = group * kRowTile + me;
      float* rec = kTree && p.partial >= 0 ? a.partial + (size_t)p.partial * partial_words<kRows, kDim>() : nullptr;
      const bool mend = *dirty >= pieces;  // a later piece's: nothing to add here, which does no harm
#pragma unroll
      for (int c = 0; c < kDim; c += 32) {
        uint32_t v[32];
        if (p.tile0 < tile1) {
          tmem_ld32(tl + C::kOCol + c, v);
          tmem_wait(v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
        if (!there) continue;
        if (mend) {
          // A weight is positive: what is not finite passes through the sum as it is.
          for (uint32_t key = max(p.tile0, blind(p.row_tile * kRows)) * kKeys; key < min(tile1 * kKeys, s.len); ++key) {
            if (!view.sees(key)) continue;
            const T* from;
            if (kTree) {
              const uint32_t page = a.tables[(uint64_t)p.seq * a.table_width + key / a.cache.page_size];
              if (page >= a.cache.pages) continue;
              from = reinterpret_cast<const T*>(a.cache.v) +
                     (((uint64_t)page * a.cache.kv_heads + p.head) * a.cache.page_size + key % a.cache.page_size) * kDim;
            } else {
              from = static_cast<const T*>(a.v.data) + (uint64_t)(s.kv0 + key) * a.v.row_stride +
                     (uint64_t)p.head * a.v.head_stride;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float x = (float)from[c + i];
              if (!(fabsf(x) < INFINITY)) v[i] = __float_as_uint(__uint_as_float(v[i]) + x);
            }
          }
        }
        if (rec) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(rec + in_tile * kDim + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float y[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) y[u] = __fmul_rn(__uint_as_float(v[i + u]), inv);
            *reinterpret_cast<uint4*>(out + c + i) = Elements<T>::store(y);
          }
        }
      }
      if (there && rec) {
        rec[kRows * kDim + in_tile] = m == -INFINITY ? m : m - F::kRaise;
        rec[kRows * kDim + kRows + in_tile] = l;
      }
    }
  }

  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (*abort_flag && tid == 0) mark_timeout();
  if (warp == 0) tmem_dealloc(*tmem_slot, C::kCols);
}

template <class T, int kDim, int kGroups, bool kTree>
uint32_t launch(const AttnArgs& a, cudaStream_t s) {
  using C = Tc<kDim, kGroups>;
  auto kernel = attention_tc_kernel<T, kDim, kGroups, kTree>;
  static std::atomic<uint64_t> configured{0};
  if (attribute_needed(configured)) {
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::bytes(PB_MAX_SEQS)));
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    attribute_done(configured);
  }
  Maps maps{};
  uint32_t st = kTree ? cache_maps<T>(a, kDim, kKeys, &maps) : rows_maps<T>(a, kDim, kKeys, &maps);
  if (st) return st;
  const uint32_t grid = kTree ? tree_ctas(C::kCtas) : (a.q_rows * a.group / C::kRows + a.seqs) * a.kv_heads;
  kernel<<<grid, C::kThreads, C::bytes(a.seqs), s>>>(a, maps);
  PB_CUDA(cudaGetLastError());
  return kTree ? launch_combine<T, kDim, C::kRows, kKeys, kLeast>(a, grid, s) : PB_OK;
}

// Three row tiles a CTA where the rows of a sequence and key head fill two on average.
bool wide(uint32_t head_dim, uint64_t rows, uint32_t seqs) {
  return head_dim == 64 && rows >= 2ull * kRowTile * seqs;
}

template <class T, bool kTree>
uint32_t by_size(const AttnArgs& a, uint32_t head_dim, cudaStream_t s) {
  if (head_dim == 128) return launch<T, 128, 1, kTree>(a, s);
  return wide(head_dim, (uint64_t)a.q_rows * a.group, a.seqs) ? launch<T, 64, 3, kTree>(a, s)
                                                              : launch<T, 64, 1, kTree>(a, s);
}

}  // namespace

uint32_t tc_prompt(const AttnArgs& a, uint32_t type, uint32_t head_dim, cudaStream_t s) {
  return type == PB_TYPE_F16 ? by_size<__half, false>(a, head_dim, s) : by_size<__nv_bfloat16, false>(a, head_dim, s);
}

uint64_t tc_tree_words(uint32_t head_dim, uint32_t rows, uint32_t seqs) {
  // CTAs x rows: three row tiles have one CTA per SM, one has two
  return wide(head_dim, rows, seqs) ? (uint64_t)tree_ctas(1) * 2 * 3 * kRowTile * (head_dim + 2)
                                    : (uint64_t)tree_ctas(2) * 2 * kRowTile * (head_dim + 2);
}

uint32_t tc_tree(const AttnArgs& a, uint32_t type, uint32_t head_dim, cudaStream_t s) {
  return type == PB_TYPE_F16 ? by_size<__half, true>(a, head_dim, s) : by_size<__nv_bfloat16, true>(a, head_dim, s);
}

uint32_t tc_status() { return take_status(); }

}  // namespace paged
}  // namespace pb
