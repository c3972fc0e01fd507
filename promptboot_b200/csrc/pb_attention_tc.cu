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
// Warps: 0..3 softmax, one row per thread (TMEM lane = row); 4 issues the MMAs;
// 5 brings K and V tiles by TMA (128-byte swizzle) into rings of kStages, and Q, as soon
// as its place is free, so that a unit's first scores are formed under the weights and
// the way out of the one before (24 ragged prompts: 163 -> 144 us).  S has two
// buffers in TMEM, P takes the place of the upper half of the scores it comes from: the
// scores of tile j + 2 go out when the products of tile j are done, a tile ahead of
// their softmax, which therefore seldom waits.  256 TMEM columns, so two CTAs share an
// SM and one's products run under the other's exponentials.
//
// Prompts: a CTA that is done cancels one that has not begun and takes its unit, so that
// the start of a CTA is paid once an SM and the longest units do not end last.
//
// Bound by the softmax warps, 750 cycles per scheduler for 64 keys of a row tile where
// the exponentials (16 a cycle and SM) need 512.  No unit is full meanwhile (issue 47%,
// exponential unit 60%, tensor pipe 33%, prompt of 8192 at heads of 64); two, three and
// four softmax warps per scheduler measured the same, 0.47 to 0.55 instructions a cycle.
// One prompt of 16384 (14 heads of 64): 0.61 ms alone, 784 TFLOP/s, 670 us where calls
// follow one another; one of 4096 at 32 heads of 128: 125 us alone, 1100 TFLOP/s.  Three
// row tiles a CTA that share the key tiles gained 5% there and lost as much on ragged
// batches; four CTAs an SM with one score buffer each, and weights formed with the
// maximum of the tile before, measured the same or worse.
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

constexpr int kThreads = 192;
constexpr int kRows = 128;
constexpr int kLeast = 2;

template <int kDim>
struct Tc {
  static constexpr int kKeys = 64;
  static constexpr int kStages = kDim == 64 ? 4 : 2;
  static constexpr int kHalves = kDim / 64;           // 128-byte column blocks of a row
  static constexpr int kQBlock = kRows * 128;
  static constexpr int kBlock = kKeys * 128;          // one column block of a K or V tile
  static constexpr int kTile = kHalves * kBlock;
  static constexpr int kKOff = kHalves * kQBlock;
  static constexpr int kVOff = kKOff + kStages * kTile;
  static constexpr int kBarOff = kVOff + kStages * kTile;
  static constexpr int kBars = 4 * kStages + 11;
  static constexpr int kPrefixOff = kBarOff + kBars * 8 + 24;
  static constexpr int kOCol = 2 * kKeys;             // S and P: [0, 64) and [64, 128)
  static constexpr int kCols = 256;
  static_assert(kOCol + kDim <= kCols, "TMEM columns");
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
// Asks for the index of a CTA of this launch that has not begun, which then never does
// (16 bytes at `to`, completing on bar); and what the answer was.
__device__ __forceinline__ void cancel_one(uint32_t leader, uint4* to, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %2, 0;\n\t"
      "@e clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n\t}"
      ::"r"(smem_u32(to)), "r"(smem_u32(bar)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ bool cancelled(const uint4* answer, uint32_t& cta) {
  uint32_t is, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, h;\n\t}"
      : "=r"(is), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  cta = x;
  return is != 0;
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

// Turns the four words of each of four neighbouring lanes: lane j's w[i] becomes lane
// i's w[j].
__device__ __forceinline__ void across_quads(uint4 (&w)[4], int lane) {
  auto swap = [&](uint4& low, uint4& high, int with) {
    const bool up = lane & with;
    uint4 x = up ? low : high;
    x.x = __shfl_xor_sync(0xffffffffu, x.x, with);
    x.y = __shfl_xor_sync(0xffffffffu, x.y, with);
    x.z = __shfl_xor_sync(0xffffffffu, x.z, with);
    x.w = __shfl_xor_sync(0xffffffffu, x.w, with);
    (up ? low : high) = x;
  };
  swap(w[0], w[1], 1);
  swap(w[2], w[3], 1);
  swap(w[0], w[2], 2);
  swap(w[1], w[3], 2);
}

template <class T, int kDim, bool kTree>
__global__ void __launch_bounds__(kThreads, 2)
attention_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Maps maps) {
  using C = Tc<kDim>;
  using F = Format<T>;
  constexpr int kKeys = C::kKeys, kStages = C::kStages, kHalves = C::kHalves;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* q_full = v_empty + kStages;
  uint64_t* p_full = q_full + 1;  // one per score buffer: a warp may be a tile ahead of another
  uint64_t* o_full = p_full + 2;  // O holds the tile's products, its P is free
  uint64_t* done = o_full + 1;    // O holds the piece's
  uint64_t* s_full = done + 1;
  uint64_t* unit_full = s_full + 2;  // prompts: the next unit is known
  uint64_t* unit_empty = unit_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(unit_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // Of four pieces in turn, the last with a value that was taken out: a warp may be in a
  // piece while another ends the one before, or, where that one had no tiles and so made
  // no warp wait for another, the one before that.
  volatile int* dirty = abort_flag + 1;
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + C::kPrefixOff);

  if (kTree) pdl_trigger();
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  work_prefix<kTree, kRows, kKeys, kThreads>(a, prefix);
  const uint32_t total = prefix[a.seqs - 1];
  uint32_t next, end;
  if (kTree) {
    const Share<kLeast> share(total, gridDim.x);
    if (total == 0 || blockIdx.x >= share.runs) {
      if (tid == 0) note_join<kRows, kKeys>(a, prefix, share, blockIdx.x);
      return;
    }
    next = share.start(blockIdx.x);
    end = share.start(blockIdx.x + 1);
  } else {
    if (blockIdx.x >= total) return;
    next = blockIdx.x;
    end = next + 1;
  }

  if (warp == 4) tmem_alloc(tmem_slot, C::kCols);
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(q_full, 32);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(&p_full[0], kRows);
    mbar_init(&p_full[1], kRows);
    mbar_init(o_full, 1);
    mbar_init(done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&unit_full[i], 1);
      mbar_init(&unit_empty[i], kThreads / 32);
    }
    *abort_flag = 0;
    for (int i = 0; i < 4; ++i) dirty[i] = 0;
    fence_barrier_init();
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = *tmem_slot;

  // The CTA's pieces, decoded alike by every role.  Prompts: one unit after another, of
  // those that no CTA has begun, by cancelling the launch of its CTA; asked for while the
  // unit before is worked on.
  __shared__ alignas(16) uint4 answer[2];
  Sequence s;
  uint32_t rows;
  int unit = 0;
  bool have = true;
  auto take = [&](Piece& p) { take_piece<kTree, kRows, kKeys>(a, prefix, blockIdx.x, next, end, p, s, rows); };
  auto further = [&] {
    if (kTree) return next < end;
    const int slot = unit & 1;
    if (!wait_soon(&unit_full[slot], (unit >> 1) & 1, abort_flag)) return false;
    const bool more = cancelled(&answer[slot], next);
    fence_async_smem();  // read before the next answer is written
    __syncwarp();
    if (lane == 0) mbar_arrive(&unit_empty[slot]);
    ++unit;
    return more && next < total;
  };

  int k_brought = 0, v_brought = 0, o_commits = 0;  // tiles, for the way out

  if (warp == 5) {
    const uint32_t leader = elect_one();
    const uint32_t size = kTree ? min(a.cache.page_size, (uint32_t)kKeys) : kKeys;  // keys of a box
    const uint32_t ka = smem_u32(smem) + C::kKOff, va = smem_u32(smem) + C::kVOff;
    int q = 0;  // tiles so far
    bool stop = false;
    int asked = 0;
    const uint32_t inverse = 0xffffffffu / a.group + 1;  // x / group of x below 2048
    // Sends for a piece's rows of Q, eight lanes to 128 bytes of a row.
    auto bring_q = [&](const Piece& p) {
      const uint32_t first = p.row_tile * kRows, token0 = first / a.group, rest = first % a.group;
      const T* from = static_cast<const T*>(a.q.data) + (uint64_t)(s.q0 + token0) * a.q.row_stride +
                      (uint64_t)(p.head * a.group) * a.q.head_stride + lane % 8 * 8;
      const uint32_t to = smem_u32(smem);
#pragma unroll 4
      for (uint32_t r = lane / 8; r < kRows; r += 4) {
        const uint32_t x = rest + r, t = a.group == 1 ? x : __umulhi(x, inverse), h = x - t * a.group;
        const bool there = first + r < rows;  // else zeros
        const T* row = from + (uint64_t)t * a.q.row_stride + (uint64_t)h * a.q.head_stride;
#pragma unroll
        for (int c = 0; c < kHalves; ++c)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                           to + c * C::kQBlock + r * 128 + ((lane % 8) ^ (r % 8)) * 16),
                       "l"(there ? static_cast<const void*>(row + c * 64) : a.q.data), "r"(there ? 16 : 0)
                       : "memory");
      }
    };
    for (; have && !stop; have = further()) {
      Piece p;
      take(p);
      if (!kTree) {
        if (!wait_soon(&unit_empty[unit & 1], ((unit >> 1) & 1) ^ 1, abort_flag)) break;
        expect_tx(leader, &unit_full[unit & 1], 16);
        cancel_one(leader, &answer[unit & 1], &unit_full[unit & 1]);
        asked = unit + 1;
      }
      auto boxes = [&](uint32_t tile) { return min((uint32_t)kKeys / size, ceil_div(s.len - tile * kKeys, size)); };
      auto page_of = [&](uint32_t tile) {  // of box `lane` of a tile
        const uint32_t key = tile * kKeys + lane * size;
        return kTree && tile < p.tile1 && (uint32_t)lane < boxes(tile)
                   ? (int)a.tables[(uint64_t)p.seq * a.table_width + key / a.cache.page_size] : 0;
      };
      int page = page_of(p.tile0);
      if (p.tile0 < p.tile1) {  // Q takes its place after the last scores of the piece before
        if (q > 0 && !wait_soon(&k_empty[(q - 1) % kStages], ((q - 1) / kStages) & 1, abort_flag)) break;
        bring_q(p);
      }
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
        if (tile == p.tile0) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_async_smem();
          mbar_arrive(q_full);
        }
        if (!wait_soon(&v_empty[st], ((q / kStages) & 1) ^ 1, abort_flag)) { stop = true; break; }
        bring(va + st * C::kTile, &maps.v, maps.v_step, &v_full[st]);
        v_brought = q + 1;
        page = ahead;
      }
    }
    if (kTree && lane == 0)  // under the last tiles of the others
      note_join<kRows, kKeys>(a, prefix, Share<kLeast>(total, gridDim.x), blockIdx.x);
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (*abort_flag) {  // every copy and answer lands before the CTA may exit
      if (asked) wait_drain(&unit_full[(asked - 1) & 1], ((asked - 1) >> 1) & 1, 50000000ull);
      for (int i = max(0, k_brought - kStages); i < k_brought; ++i)
        wait_drain(&k_full[i % kStages], (i / kStages) & 1, 50000000ull);
      for (int i = max(0, v_brought - kStages); i < v_brought; ++i)
        wait_drain(&v_full[i % kStages], (i / kStages) & 1, 50000000ull);
    }
    __syncwarp();
  } else if (warp == 4) {
    const uint32_t leader = elect_one();
    constexpr uint32_t kBase = (1u << 4) | (F::kCode << 7) | (F::kCode << 10) | ((uint32_t)(kRows >> 4) << 24);
    constexpr uint32_t kQk = kBase | ((uint32_t)(kKeys >> 3) << 17);
    constexpr uint32_t kPv = kBase | ((uint32_t)(kDim >> 3) << 17) | (1u << 16);  // V is N-major
    const uint32_t qa = smem_u32(smem), ka = qa + C::kKOff, va = qa + C::kVOff;
    int q = 0, pieces = 0;  // tiles and pieces so far
    bool stop = false;
    for (; have && !stop; have = further()) {
      Piece p;
      take(p);
      const int n = (int)(p.tile1 - p.tile0);
      if (n <= 0) continue;
      auto scores = [&](int t) {  // S = Q K^T
        const int st = t % kStages;
        if (!wait_soon(&k_full[st], (t / kStages) & 1, abort_flag)) return false;
        tc_after_sync();
#pragma unroll
        for (int j = 0; j < kDim / 16; ++j)
          mma_ss(leader, tmem + (t & 1) * kKeys, desc128(qa + j / 4 * C::kQBlock + j % 4 * 32, 16),
                 desc128(ka + st * C::kTile + j / 4 * C::kBlock + j % 4 * 32, 16), kQk, j > 0);
        commit_to(leader, &s_full[t & 1]);
        commit_to(leader, &k_empty[st]);
        return true;
      };
      if (!wait_soon(q_full, pieces & 1, abort_flag) || !scores(q) || (n > 1 && !scores(q + 1))) break;
      ++pieces;
      for (int i = 0; i < n; ++i, ++q) {
        const int st = q % kStages;
        if (!wait_soon(&p_full[q & 1], (q >> 1) & 1, abort_flag) || !wait_soon(&v_full[st], (q / kStages) & 1, abort_flag)) {
          stop = true;
          break;
        }
        tc_after_sync();
#pragma unroll
        for (int j = 0; j < kKeys / 16; ++j)
          mma_ts(leader, tmem + C::kOCol, tmem + (q & 1) * kKeys + kKeys / 2 + j * 8,
                 desc128(va + st * C::kTile + j * 2048, C::kBlock), kPv, i > 0 || j > 0);
        commit_to(leader, o_full);
        commit_to(leader, &v_empty[st]);
        if (i + 1 == n) commit_to(leader, done);
        o_commits = q + 1;
        // The scores of the tile after the next take the place of this P, once it has
        // been read.
        if (!wait_soon(o_full, q & 1, abort_flag) || (i + 2 < n && !scores(q + 2))) {
          stop = true;
          break;
        }
      }
    }
    if (*abort_flag && o_commits) wait_drain(o_full, (o_commits - 1) & 1, 50000000ull);  // issued MMAs end
    __syncwarp();
  } else {
    const uint32_t tl = tmem + ((uint32_t)(warp * 32) << 16);  // this warp's lanes
    int q = 0, pieces = 0, walked = 0;  // tiles; pieces, and those with tiles
    bool stop = false;
    for (; have && !stop; have = further()) {
      Piece p;
      take(p);
      ++pieces;
      const uint32_t row = p.row_tile * kRows + tid, token = row / a.group;
      const uint32_t head = p.head * a.group + row % a.group;
      const bool there = row < rows;
      // Rows past the last see everything: zeros times finite or other keys, never stored.
      const RowView view = there ? row_view<kTree>(a, s, token) : RowView{0xffffffffu, 0ull};
      float m = -INFINITY;          // the maximum in use, in powers of two
      uint64_t l2[2] = {0, 0};      // the sum of weights, in four parts
      // Tiles from here on hold a key that some row does not see.
      const uint32_t mask0 = (kTree ? s.context : row_view<false>(a, s, p.row_tile * kRows / a.group).all) / kKeys;
      for (uint32_t tile = p.tile0; tile < p.tile1; ++tile, ++q) {
        const uint32_t key0 = tile * kKeys;
        const bool masked = tile >= mask0;
        const uint32_t sc = tl + (q & 1) * kKeys;
        if (!wait_soon(&s_full[q & 1], (q >> 1) & 1, abort_flag)) { stop = true; break; }
        tc_after_sync();
        uint32_t v[2][32];
        tmem_ld32(sc, v[0]);
        tmem_ld32(sc + 32, v[1]);
        tmem_wait(v[0]);
        tmem_wait(v[1]);
        if (masked) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t seen = seen32(view, key0 + 32 * c);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[c][i] = (seen >> i) & 1 ? v[c][i] : 0xff800000u;  // -inf
          }
        }
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            t[u] = max_nan(t[u], __uint_as_float(v[i / 32][i % 32 + 2 * u]),
                           __uint_as_float(v[i / 32][i % 32 + 2 * u + 1]));
        const float top = __fmul_rn(max_nan(max_nan(t[0], t[1], t[2]), t[3], t[3]), a.scale_log2);
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
          if (!wait_soon(o_full, (q - 1) & 1, abort_flag)) { stop = true; break; }
          tc_after_sync();
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
        // One exponential in eight through the polynomial (one in four took 626 us for the
        // prompt of 16384 where this takes 621 and none 638); all through the unit where
        // keys are masked, whose weight has to be zero.
        auto weigh = [&](auto mixed) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              uint64_t y = fma2(pk_u(v[c][i], v[c][i + 1]), scale2, base2);
              y = decltype(mixed)::value && i % 16 == 14 ? exp2_poly<F::kDegree>(y) : exp2_pair(y);
              l2[i / 2 & 1] = add2(l2[i / 2 & 1], y);
              float y0, y1;
              unpk(y, y0, y1);
              w[i / 2] = Elements<T>::pair(y0, y1);
            }
            tmem_st16(sc + kKeys / 2 + 16 * c, w);  // over scores that have been read
          }
        };
        if (masked) weigh(std::false_type{});
        else weigh(std::true_type{});
        if (masked) {
          // Value rows of this tile, half a row per thread: zero past the keys, and without
          // what is not finite.
          if (!wait_soon(&v_full[q % kStages], (q / kStages) & 1, abort_flag)) { stop = true; break; }
          static_assert(2 * kKeys == kRows, "two threads to a value row");
          const int key = tid % kKeys;
          if (clean_value_row<F, kDim, C::kBlock, 2>(smem + C::kVOff + (q % kStages) * C::kTile, key, tid / kKeys,
                                                     key0 + key >= s.len))
            dirty[pieces & 3] = pieces;
          fence_async_smem();
        }
        tmem_wait_st();
        tc_before_sync();
        mbar_arrive(&p_full[q & 1]);
      }
      if (stop) break;

      // The piece is done: O / l, or O with its maximum and sum.
      if (p.tile0 < p.tile1) {
        if (!wait_soon(done, walked & 1, abort_flag)) break;
        ++walked;
        tc_after_sync();
      }
      float part[4];
      unpk(l2[0], part[0], part[1]);
      unpk(l2[1], part[2], part[3]);
      // No weight where every score is -inf: the polynomial gives those 2^-126 instead of none.
      const float l = m == -INFINITY ? 0.f : (part[0] + part[1]) + (part[2] + part[3]);
      const float inv = l == 0.f ? 0.f : __frcp_rn(l);
      T* out = static_cast<T*>(a.out.data) + (uint64_t)(s.q0 + token) * a.out.row_stride +
               (uint64_t)head * a.out.head_stride;
      float* rec = kTree && p.partial >= 0 ? a.partial + (size_t)p.partial * partial_words<kRows, kDim>() : nullptr;
      T* quad[4];  // the rows of four neighbouring threads, whose stores then fill 64 bytes of a row
#pragma unroll
      for (int i = 0; i < 4; ++i)
        quad[i] = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, (unsigned long long)out, (lane & ~3) + i));
      const bool mend = dirty[pieces & 3] == pieces;
#pragma unroll
      for (int c = 0; c < kDim; c += 32) {
        uint32_t v[32];
        if (p.tile0 < p.tile1) {
          tmem_ld32(tl + C::kOCol + c, v);
          tmem_wait(v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
        if (mend && there) {
          // A weight is positive: what is not finite passes through the sum as it is.
          for (uint32_t key = max(p.tile0, mask0) * kKeys; key < min(p.tile1 * kKeys, s.len); ++key) {
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
          if (there) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(rec + tid * kDim + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
        } else {
          uint4 w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float y[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) y[u] = __fmul_rn(__uint_as_float(v[8 * i + u]), inv);
            w[i] = Elements<T>::store(y);
          }
          across_quads(w, lane);  // word `lane % 4` of the quad's four rows
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row - lane % 4 + i < rows) *reinterpret_cast<uint4*>(quad[i] + c + lane % 4 * 8) = w[i];
        }
      }
      if (there && rec) {
        rec[kRows * kDim + tid] = m == -INFINITY ? m : m - F::kRaise;
        rec[kRows * kDim + kRows + tid] = l;
      }
    }
  }

  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (*abort_flag && tid == 0) mark_timeout();
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (warp == 4) tmem_dealloc(tmem, C::kCols);
}

template <class T, int kDim, bool kTree>
uint32_t launch(AttnArgs a, uint32_t grid, cudaStream_t s) {
  using C = Tc<kDim>;
  auto kernel = attention_tc_kernel<T, kDim, kTree>;
  static std::atomic<uint64_t> configured{0};
  if (attribute_needed(configured)) {
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::bytes(PB_MAX_SEQS)));
    PB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    attribute_done(configured);
  }
  Maps maps{};
  uint32_t st = kTree ? cache_maps<T>(a, kDim, C::kKeys, &maps) : rows_maps<T>(a, kDim, C::kKeys, &maps);
  if (st) return st;
  if (kTree) place_workspace(a, grid, kRows, kDim);
  kernel<<<grid, kThreads, C::bytes(a.seqs), s>>>(a, maps);
  PB_CUDA(cudaGetLastError());
  return kTree ? launch_combine<T, kDim, kRows>(a, grid, s) : PB_OK;
}

}  // namespace

uint32_t tc_prompt(const AttnArgs& a, uint32_t type, uint32_t head_dim, cudaStream_t s) {
  const uint32_t grid = (a.q_rows * a.group / kRows + a.seqs) * a.kv_heads;
  if (type == PB_TYPE_F16)
    return head_dim == 64 ? launch<__half, 64, false>(a, grid, s) : launch<__half, 128, false>(a, grid, s);
  return head_dim == 64 ? launch<__nv_bfloat16, 64, false>(a, grid, s)
                        : launch<__nv_bfloat16, 128, false>(a, grid, s);
}

uint64_t tc_tree_words(uint32_t head_dim) { return tree_words(tree_ctas(2), kRows, head_dim); }

uint32_t tc_tree(const AttnArgs& a, uint32_t type, uint32_t head_dim, cudaStream_t s) {
  const uint32_t grid = tree_ctas(2);
  if (type == PB_TYPE_F16)
    return head_dim == 64 ? launch<__half, 64, true>(a, grid, s) : launch<__half, 128, true>(a, grid, s);
  return head_dim == 64 ? launch<__nv_bfloat16, 64, true>(a, grid, s) : launch<__nv_bfloat16, 128, true>(a, grid, s);
}

uint32_t tc_timeouts(cudaStream_t s, uint32_t* count) { return add_timeouts(s, count); }

}  // namespace paged
}  // namespace pb
