// Attention of chunks of new tokens over paged keys and values (every
// sequence that paged_decode.cu does not take) on the tcgen05 tensor cores.
//
// A CTA works on pairs of row tiles: the G query heads of a KV head times
// 128 / G consecutive queries are the M = 128 rows of a tile (query-major), so
// every key tile serves the whole group and 2 * 128 / G queries. Per key tile j
// of 128 keys and row tile x in {0, 1}:
//   S_x = Q_x K_j^T     M128 N128, FP32 in tensor memory
//   softmax             thread r of warpgroup x owns row r, its tensor-memory
//                       lane: reads S_x, masks, writes P_x (fp16) over it
//   O_x += P_x V_j      M128 N = dim, A = P_x from tensor memory, B = V_j
//                       MN-major straight from the TMA tile
// While the softmax of one row tile runs, the tensor cores work for the other:
// the issue order is P_0 V, Q_0 K', P_1 V, Q_1 K', ... A row tile's next S
// overwrites its P: tcgen05.mma of one thread run in order.
// FP32 queries are two fp16 terms (two MMAs for S, two terms of P, which fill
// the 128 columns of S, two MMAs for O): 22 bits where a 16-bit type has one.
// Rows are scaled to fp16's range by a power of two each first.
// A row's probabilities are 2^(x - m) with a reference m that trails the
// running maximum: 2^7 for the maximum when m moves, 2^15 at most before it
// moves again, so it (and with it O in tensor memory) moves rarely and
// small probabilities stay clear of fp16's subnormals. Where a step of FP32 is
// no longer small against these exponents (m past 2^22) a score is rounded to
// FP32 before m is taken from it, as the maximum was: one fused operation would
// leave the rounding of the maximum in the exponent, and a probability of 2^64.
// Masked keys. A key that a row does not see has probability 0, but 0 times a
// NaN or an infinity in V would still reach the row's sums. In tiles where
// some row sees less than all keys (the diagonal, a window's edge, the last
// page's tail) a warp of its own therefore clears, between the copy and P V,
// the rows that no row of the pair sees and the values that are not finite;
// rows that do see such a value get it added at the end.
// Blocks take equal shares of the batch's (row tile pair, KV head, key tile)
// units (paged_plan.cuh), so one long history is split over all SMs. Warps:
// 0-3 and 4-7 softmax and epilogue (a warp loads, converts and writes its own
// 32 rows, a row at a time over the lanes), 8 TMA, 9 tensor memory and (one
// thread) every MMA, 10 the clearing, 11 works out the segments ahead of the
// others. Every wait is bounded.
// Two chunks of 2048 bf16 rows at depth 16384 (504 GFLOP): 525 to 547 us, 0.92
// to 0.96 PFLOP/s, the clock falling under the power limit. Neither the tensor
// cores nor the special function units are full (each busy for 42 % of two
// chunks of 1000 rows at depth 5000): the chain of S, softmax and P V of two
// row tiles is. A polynomial on the FMA pipe for an eighth of the exponentials
// gained 1 % and cost bits, so there is none. 512 FP32 rows at depth 8192 (two
// terms, 71 GFLOP as such): 90 us with the merge, of which 60 us are key tiles,
// the rest the single-token kernel before it, the plan, the queries'
// conversion, O's moves and the merge.
#include <type_traits>

#include "kernels.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "tcgen05.cuh"
#include "tensor_map.hpp"

namespace lfm3 {
namespace {

constexpr int kThreads = 12 * 32;
constexpr uint32_t kColS = 128, kColO = 256, kColumns = 512;
constexpr uint32_t kSlab = 128 * 128;  // bytes of [128 rows][64 dims]
constexpr int kPlanned = 4;            // segments worked out ahead
// key tiles in the time that a segment takes beyond its tiles (2, 3 and 5 for
// two terms, 4 and 8 for one: up to 5 % and 17 % slower)
template <int TERMS>
constexpr int kSegmentUnits = TERMS == 2 ? 4 : 6;
// exponents (base 2) of a row's largest probability: when the reference
// moves, and when it has to move again
constexpr float kTopMoved = 7.0F, kTopLimit = 15.0F;
constexpr float kLargeScore = 4194304.0F;  // its step is 2^-1
// Tensor-memory sums drop what falls below their last bit, always towards
// zero: each step of 16 keys and term loses about 2^-24.5 of O. Every so many
// key tiles O therefore moves to the block's slot, where it is added up with
// rounding. FP32 rows: every 4 tiles (512 rows at depth 8192: 5.3e-6 off in
// the 2-norm and 83 us without, 1.6e-6 and 94 us with; every 2 tiles 1.0e-6
// and 101 us; repeated). fp16 rows: before the loss nears their own half step.
// bf16 rows would take more than 2^20 keys a block to notice, and never do.
template <typename T>
constexpr int kFlushTiles = 1 << 30;
template <>
constexpr int kFlushTiles<float> = 4;
template <>
constexpr int kFlushTiles<__half> = 256;

template <int DIM, int TERMS>
struct __align__(1024) ChunkSmem {
  static constexpr int kSlabs = DIM / 64;
  static constexpr int kTile = kSlabs * kSlab;
  static constexpr int kStages =
      DIM == 128 ? (TERMS == 2 ? 3 : 5) : (TERMS == 2 ? 8 : 10);
  uint8_t q[2][TERMS][kTile];  // and the epilogue's rows
  uint8_t kv[kStages][kTile];  // K_0 V_0 K_1 V_1 ... in turn
  // landed; landed and cleared; free again
  uint64_t kv_full[kStages], kv_ready[kStages], kv_empty[kStages];
  uint64_t q_full[2], q_free[2], s_full[2], p_full[2][3], o_full[2], idle;
  uint64_t seg_full[kPlanned], seg_empty[kPlanned];
  ChunkSegment seg[kPlanned];
  uint32_t tmem;
  int odd_values;  // a value that is not finite was cleared
};

// Whether one of a word's two fp16 values is infinite or NaN.
__device__ __forceinline__ bool not_finite2(uint32_t u) {
  return (((u & 0x7C007C00u) + 0x04000400u) & 0x80008000u) != 0;
}
__device__ __forceinline__ uint32_t clear_not_finite(uint32_t u) {
  if ((u & 0x7C00u) == 0x7C00u)
    u &= 0xFFFF0000u;
  if ((u & 0x7C000000u) == 0x7C000000u)
    u &= 0x0000FFFFu;
  return u;
}

// Maxima of N rows over groups of LANES lanes, N values a lane: the lanes trade
// halves of their rows (N - 1 shuffles, not N log LANES). Lane `part` of a
// group gets the maximum of row part / (LANES / N).
template <int N, int LANES>
__device__ __forceinline__ float group_max(const float (&v)[N], int part) {
  if constexpr (LANES == 1) {
    static_assert(N == 1);
    return v[0];
  } else {
    constexpr int o = LANES / 2, n = N > 1 ? N / 2 : 1;
    float w[n];
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const float keep = part & o ? v[N - n + k] : v[k];
      const float give = part & o ? v[k] : v[N - n + k];
      w[k] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
    return group_max<n, o>(w, part);
  }
}

// What a pair of row tiles sees: rows are the sequence's new rows q0 .. qlast.
// Every row sees keys all_lo .. all_hi, some row any_lo .. any_hi.
struct PairRange {
  int q0, qlast, base, all_lo, all_hi, any_lo, any_hi;
  __device__ PairRange(const ChunkSegment& g, int QB, int window) {
    q0 = g.pair * 2 * QB;
    qlast = min(g.q.n, q0 + 2 * QB) - 1;
    base = g.q.length - g.q.n;
    all_hi = base + q0;
    any_hi = base + qlast;
    // (idle rows have negative numbers: compared before the subtraction)
    const auto oldest = [&](int own) {
      return window > 0 && own >= window ? own - window + 1 : 0;
    };
    all_lo = oldest(base + qlast);
    any_lo = oldest(base + q0);
  }
  // some row sees less than the whole tile
  __device__ bool edge(int key0) const {
    return key0 + kChunkKeys - 1 > all_hi || key0 < all_lo;
  }
};

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads, 1)
    paged_chunk_kernel(const __grid_constant__ PagedAttentionArgs a) {
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  using Smem = ChunkSmem<DIM, TERMS>;
  constexpr int kStages = Smem::kStages, kSlabs = Smem::kSlabs;
  constexpr uint32_t kIdescS = tc::f16_idesc(128, 128);
  constexpr uint32_t kIdescO = tc::f16_idesc(128, DIM, true);
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int kvh = a.t.kv_heads, group = a.heads / kvh;
  const int QB = chunk_queries(group);
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.kv_full[i], 1);
      mbar_init(&s.kv_ready[i], 1);
      mbar_init(&s.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 4);
      mbar_init(&s.q_free[i], 4);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i][0], 4);
      mbar_init(&s.p_full[i][1], 4);
      mbar_init(&s.p_full[i][2], 4);
      mbar_init(&s.o_full[i], 1);
    }
    for (int i = 0; i < kPlanned; ++i) {
      mbar_init(&s.seg_full[i], 1);
      mbar_init(&s.seg_empty[i], 11);  // every other warp
    }
    mbar_init(&s.idle, 1);
    s.odd_values = 0;
    fence_barrier_init();
    prefetch_map(&a.kmap);
    prefetch_map(&a.vmap);
  }
  if (warp == 9)
    tc::alloc(&s.tmem, kColumns);
  grid_dependency_wait();
  allow_dependents();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = s.tmem;
  bool ok = true;
  ChunkSegment g;
  uint32_t planned = 0;
  // The next segment (warp-wide): false at the end of the block's share. A
  // barrier's phase is the parity of its completed uses.
  const auto next_segment = [&]() {
    const uint32_t i = planned % kPlanned;
    ok = ok && __all_sync(0xffffffffu,
                          mbar_wait(&s.seg_full[i], (planned / kPlanned) & 1,
                                    kErrPagedWait));
    if (!ok)
      return false;
    g = s.seg[i];
    __syncwarp();
    if (lane == 0)
      mbar_arrive(&s.seg_empty[i]);
    ++planned;
    return g.count > 0;
  };

  if (warp == 11) {
    // ---- the block's segments, then one with count 0
    PagedLine<ChunkUnits> line(
        a.t, ChunkUnits{group, a.window, 1, kSegmentUnits<TERMS>});
    const int64_t share = chunk_plan(line);
    if (line.broken && blockIdx.x == 0)
      report_error(kErrPagedTable);
    const int64_t total = line.total * kvh;
    const int64_t begin = share * blockIdx.x, end = min(begin + share, total);
    PagedRecord record{0, 0, 0, 0, 0, 0};
    int64_t at = begin;
    for (bool more = true; more && ok; ++planned) {
      more = chunk_segment(line, at, end, g);
      if (more && g.count == 0) {  // the empty places behind a stretch
        at += g.units;
        more = chunk_segment(line, at, end, g);
      }
      if (!more)
        g.count = g.units = 0;
      g.slot = 2 * blockIdx.x + (at > begin ? 1 : 0);
      const uint32_t i = planned % kPlanned;
      if (planned >= kPlanned)
        ok = __all_sync(0xffffffffu,
                        mbar_wait(&s.seg_empty[i],
                                  ((planned / kPlanned) - 1) & 1,
                                  kErrPagedWait));
      if (lane == 0 && ok) {
        s.seg[i] = g;
        mbar_arrive(&s.seg_full[i]);
      }
      __syncwarp();
      if (more && g.count < g.n_units && g.u0 == 0)
        record = paged_record(at, share, g.slot, g.n_units, g.q, g.pair, g.h);
      at += g.units;
    }
    if (lane == 0)
      reinterpret_cast<PagedRecord*>(
          a.chunk_part +
          size_t(2 * kChunkCtas) * 256 * (DIM + 2))[blockIdx.x] = record;
  } else if (warp == 8) {
    // ---- TMA: K and V tiles, a lane per box
    const int per = 128 / a.box_rows;  // boxes of a slab
    uint32_t loads = 0;
    while (next_segment()) {
      // page ids are read a key tile ahead of their copies
      const auto pool_row = [&](int j) {
        const int key0 = (g.lo_unit + g.u0 + j) * kChunkKeys;
        const int key = key0 + lane / kSlabs * a.box_rows;
        // (at most 16 boxes of a key tile, each with rows of the sequence)
        return j < g.count && lane < per * kSlabs && key < g.q.length
                   ? paged_row(a.t, a.t.table, g.seq, key)
                   : 0;
      };
      int next = pool_row(0);
      for (int j = 0; j < g.count && ok; ++j) {
        const int key0 = (g.lo_unit + g.u0 + j) * kChunkKeys;
        const int boxes =
            min(per, (g.q.length - key0 + a.box_rows - 1) / a.box_rows);
        int row = next;
        next = pool_row(j + 1);
        if (row < 0) {
          report_error(kErrPagedTable);
          row = 0;
        }
#pragma unroll
        for (int v = 0; v < 2; ++v, ++loads) {
          const int st = loads % kStages;
          if (loads >= kStages)
            ok = ok && __all_sync(0xffffffffu,
                                  mbar_wait(&s.kv_empty[st],
                                            ((loads / kStages) - 1) & 1,
                                            kErrPagedWait));
          if (!ok)
            break;
          if (lane == 0)
            mbar_arrive_expect_tx(&s.kv_full[st],
                                  uint32_t(boxes * kSlabs * a.box_rows) * 128);
          __syncwarp();
          if (lane < boxes * kSlabs)
            tma_load_3d(s.kv[st] + lane % kSlabs * kSlab +
                            lane / kSlabs * a.box_rows * 128,
                        v ? &a.vmap : &a.kmap, 0, row,
                        g.h * kSlabs + lane % kSlabs, &s.kv_full[st]);
        }
      }
    }
    // no copy may still be landing when the block exits
    for (uint32_t i = loads > kStages ? loads - kStages : 0; i < loads; ++i)
      mbar_wait(&s.kv_full[i % kStages], (i / kStages) & 1, kErrPagedWait);
  } else if (warp == 10) {
    // ---- clearing what masked rows must not meet in V
    uint32_t loads = 0;
    while (next_segment()) {
      const PairRange range(g, QB, a.window);
      for (int i = 0; i < 2 * g.count && ok; ++i, ++loads) {
        const int st = loads % kStages;
        ok = __all_sync(0xffffffffu,
                        mbar_wait(&s.kv_full[st], (loads / kStages) & 1,
                                  kErrPagedWait));
        if (!ok)
          break;
        const int key0 = (g.lo_unit + g.u0 + i / 2) * kChunkKeys;
        if (i % 2 && range.edge(key0)) {
          uint8_t* v = s.kv[st];
          // Few instructions: the softmax warps leave this warp few issue
          // slots. Rows lo .. hi of the tile are seen by some row of the
          // pair; the others become 0, then one maximum over everything
          // tells whether a value is not finite. A 16-byte piece's row is its
          // place by 128 bytes, whatever the swizzle does inside the row.
          const int lo = min(max(range.any_lo - key0, 0), 128);
          const int hi = min(range.any_hi - key0, 127);
          const int hidden = (lo + 127 - hi) * 8;  // pieces a slab
          for (int e = lane; e < hidden * kSlabs; e += 32) {
            const int slab = e >= hidden, i = e - slab * hidden;
            const int at16 = i < lo * 8 ? i : i - lo * 8 + (hi + 1) * 8;
            *reinterpret_cast<uint4*>(v + slab * kSlab + at16 * 16) =
                make_uint4(0, 0, 0, 0);
          }
          __syncwarp();
          __half2 top = __float2half2_rn(0.0F);
          for (int e0 = lane; e0 < 128 * kSlabs * 8; e0 += 256) {
            uint4 w[8];
#pragma unroll
            for (int b = 0; b < 8; ++b)
              w[b] = *reinterpret_cast<const uint4*>(v + (e0 + 32 * b) * 16);
#pragma unroll
            for (int b = 0; b < 8; ++b) {
              const __half2* h = reinterpret_cast<const __half2*>(&w[b]);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                top = __hmax2_nan(top, __habs2(h[k]));
            }
          }
          if (__any_sync(0xffffffffu,
                         not_finite2(*reinterpret_cast<uint32_t*>(&top)))) {
            for (int e = lane; e < 128 * kSlabs * 8; e += 32) {
              uint4* at16 = reinterpret_cast<uint4*>(v + e * 16);
              uint4 w = *at16;
              w.x = clear_not_finite(w.x);
              w.y = clear_not_finite(w.y);
              w.z = clear_not_finite(w.z);
              w.w = clear_not_finite(w.w);
              *at16 = w;
            }
            if (lane == 0)
              *reinterpret_cast<volatile int*>(&s.odd_values) = 1;
          }
          fence_proxy_async();
          __syncwarp();
        }
        if (lane == 0)
          mbar_arrive(&s.kv_ready[st]);
      }
    }
  } else if (warp == 9) {
    // ---- every MMA, issued by one lane. The softmax warps leave this warp few
    // issue slots, so what it needs is kept in uniform registers (a value of
    // a warp-wide reduction is one) and worked out before each wait.
    const bool lead = tc::elect();
    const auto uniform = [](int v) {
      return int(__reduce_max_sync(0xffffffffu, unsigned(v)));
    };
    const auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) ||
             __all_sync(0xffffffffu, mbar_wait(bar, parity, kErrPagedWait));
    };
    const uint32_t tm = uniform(tmem);
    const uint64_t qdesc = tc::sw128_desc(s.q[0][0]);
    const uint64_t kdesc = tc::sw128_desc(s.kv[0]);
    const uint64_t vdesc = tc::sw128_mn_desc(s.kv[0], kSlab);
    constexpr uint32_t kStep = Smem::kTile / 16;  // a stage, a term
    // stage and phase of the next load; uses of each row tile's barriers
    uint32_t stage = 0, phase = 0, tiles0 = 0, tiles1 = 0;
    uint32_t segment0 = 0, segment1 = 0;
    const auto advance = [&]() {
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    };
    const auto scores = [&](int x, uint32_t st) {
      const uint64_t k = kdesc + st * kStep;
      const uint64_t q = qdesc + x * TERMS * kStep;
      // the smaller term first: a step's loss goes with the sum so far
#pragma unroll
      for (int t = TERMS - 1; t >= 0; --t)
#pragma unroll
        for (int k16 = 0; k16 < DIM / 16; ++k16) {
          const int at = (k16 / 4) * (kSlab / 16) + (k16 % 4) * 2;
          tc::mma_lead(tm + x * kColS, q + t * kStep + at, k + at, kIdescS,
                       t < TERMS - 1 || k16 > 0, lead);
        }
      tc::commit_lead(&s.s_full[x], lead);
    };
    // O += P V in the pieces the softmax hands over: keys 0 .. 63, 64 .. 95
    // and 96 .. 127
    const auto consume = [&](int x, uint32_t st, uint32_t more,
                             uint32_t parity) {
      const uint64_t v = vdesc + st * kStep;
      const uint32_t p = tm + x * kColS, o = tm + kColO + x * 128;
#pragma unroll
      for (int third = 0; third < 3; ++third) {
        if (!wait(&s.p_full[x][third], parity))
          return false;
        tc::fence_after();
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
          for (int k16 = third ? 2 + 2 * third : 0; k16 < 4 + 2 * third; ++k16)
            tc::mma_ts_lead(o, p + k16 / 2 * 32 + t * 16 + k16 % 2 * 8,
                            v + k16 * 128, kIdescO,
                            t > 0 || k16 > 0 ? 1u : more, lead);
      }
      return true;
    };
    while (next_segment()) {
      const int count = uniform(g.count);
      // row tile 1 is there
      const int two = uniform(g.q.n - g.pair * 2 * QB > QB);
      ok = wait(&s.kv_ready[stage], phase) &&
           wait(&s.q_full[0], segment0 & 1) &&
           (!two || wait(&s.q_full[1], segment1 & 1));
      if (!ok)
        break;
      tc::fence_after();
      scores(0, stage);
      if (two)
        scores(1, stage);
      tc::commit_lead(&s.kv_empty[stage], lead);
      advance();
      for (int j = 0; j < count; ++j) {
        const uint32_t vs = stage, later = j % kFlushTiles<T> != 0;
        const bool more = j + 1 < count;
        ok = wait(&s.kv_ready[vs], phase);
        advance();
        const uint32_t ks = stage;
        if (more)
          ok = ok && wait(&s.kv_ready[ks], phase);
        ok = ok && consume(0, vs, later, (tiles0 + j) & 1);
        if (!ok)
          break;
        if (!two)
          tc::commit_lead(&s.kv_empty[vs], lead);
        // O is whole: at the end, and where it moves out of tensor memory
        const bool handed = !more || (j + 1) % kFlushTiles<T> == 0;
        if (handed)
          tc::commit_lead(&s.o_full[0], lead);
        if (more)
          scores(0, ks);
        if (two) {
          ok = consume(1, vs, later, (tiles1 + j) & 1);
          if (!ok)
            break;
          tc::commit_lead(&s.kv_empty[vs], lead);
          if (handed)
            tc::commit_lead(&s.o_full[1], lead);
          if (more)
            scores(1, ks);
        }
        if (more) {
          tc::commit_lead(&s.kv_empty[ks], lead);
          advance();
        }
      }
      if (!ok)
        break;
      tiles0 += count;
      ++segment0;
      if (two) {
        tiles1 += count;
        ++segment1;
      }
    }
    tc::commit_lead(&s.idle, lead);
    mbar_wait(&s.idle, 0, kErrPagedWait);
  } else {
    // ---- softmax and epilogue of row tile x: thread t owns row t
    const int x = warp / 4, t = tid % 128;
    const uint32_t lane_base = uint32_t((warp % 4) * 32) << 16;
    const uint32_t ts = tmem + lane_base + x * kColS;
    const uint32_t to = tmem + lane_base + kColO + x * 128;
    // rows over the lanes: kRowLanes lanes of 16 bytes hold one row
    constexpr bool kCanFlush = kFlushTiles<T> < 1 << 30;
    constexpr bool kHalfType = std::is_same_v<T, __half>;
    constexpr int kVec = 16 / sizeof(T), kRowLanes = DIM / kVec;
    constexpr int kRowsAtOnce = 32 / kRowLanes;
    const int sub = lane / kRowLanes, part = lane % kRowLanes;
    const int row_query = t / group, row_head = t % group;
    // a warp's lanes give up together: tensor-memory accesses are warp-wide
    const auto wait_all = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, kErrPagedWait));
    };
    uint32_t tiles = 0, segments = 0, o_uses = 0;
    while (next_segment()) {
      const PairRange range(g, QB, a.window);
      if (x == 1 && g.q.n - range.q0 <= QB)
        continue;
      const int qi = range.q0 + x * QB + row_query;
      const int head = g.h * group + row_head;
      const bool live = row_query < QB && qi < g.q.n;
      const size_t row = size_t(g.q.row0) + (live ? qi : 0);
      // the row sees keys oldest .. own
      const int own = live ? range.base + qi : -1;
      const int oldest =
          a.window > 0 && own >= a.window ? own - a.window + 1 : 0;
      float c = 1;
      {
        // ---- this warp's 32 rows of Q as fp16 terms
        // (the row tile's warps have read their rows of the last segment)
        if (segments > 0 &&
            !wait_all(&s.q_free[x], (segments - 1) & 1)) {
          ok = false;
          break;
        }
        const size_t offset = row * a.ldq + size_t(head) * DIM;
        const unsigned alive = __ballot_sync(0xffffffffu, live);
        constexpr int kBatch = kRowsAtOnce > 2 ? 32 / kRowsAtOnce : 16;
        // A power of two of its own brings each row into fp16's range (none is
        // needed for fp16 itself). The lanes of a row's group hold the scales
        // of kBatch rows, kSame lanes each.
        constexpr int kSame = kRowLanes / kBatch;
        static_assert(kSame * kBatch == kRowLanes);
#pragma unroll 1
        for (int i0 = 0; i0 < 32; i0 += kBatch * kRowsAtOnce) {
          uint4 raw[kBatch];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int r = i0 + i * kRowsAtOnce + sub;
            const size_t at =
                __shfl_sync(0xffffffffu, (unsigned long long)offset, r);
            raw[i] = make_uint4(0, 0, 0, 0);
            if (alive >> r & 1)
              raw[i] = *reinterpret_cast<const uint4*>(
                  static_cast<const T*>(a.q) + at + part * kVec);
          }
          float scales = 1;  // of row part / kSame of the lane's group
          if constexpr (!kHalfType) {
            float top[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
              float v[kVec];
              unpack16(raw[i], v, T{});
              top[i] = 0;
#pragma unroll
              for (int k = 0; k < kVec; ++k)
                top[i] = fmaxf(top[i], fabsf(v[k]));
            }
            scales = row_scale(group_max<kBatch, kRowLanes>(top, part));
            // this thread's own row: which lane holds its scale
            const int at = lane - i0;
            const float mine = __shfl_sync(
                0xffffffffu, scales,
                at % kRowsAtOnce * kRowLanes + at / kRowsAtOnce * kSame);
            if (at >= 0 && at < kBatch * kRowsAtOnce)
              c = mine;
          }
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int r = i0 + i * kRowsAtOnce + sub;
            const int piece = part * kVec / 8;
            const uint32_t off =
                (piece / 8) * kSlab +
                tc::sw128_offset((warp % 4) * 32 + r, piece % 8);
            if constexpr (kHalfType) {
              *reinterpret_cast<uint4*>(s.q[x][0] + off) = raw[i];
              continue;
            }
            const float scale =
                __shfl_sync(0xffffffffu, scales, lane - part + i * kSame);
            float v[kVec];
            uint32_t hi[kVec / 2], lo[kVec / 2];
            unpack16(raw[i], v, T{});
#pragma unroll
            for (int k = 0; k < kVec / 2; ++k) {
              const float v0 = v[2 * k] * scale, v1 = v[2 * k + 1] * scale;
              hi[k] = half2_bits(v0, v1);
              const float2 back = bits_half2(hi[k]);
              lo[k] = half2_bits(v0 - back.x, v1 - back.y);
            }
            if constexpr (TERMS == 2) {
              *reinterpret_cast<uint2*>(s.q[x][0] + off + (part & 1) * 8) =
                  make_uint2(hi[0], hi[1]);
              *reinterpret_cast<uint2*>(s.q[x][1] + off + (part & 1) * 8) =
                  make_uint2(lo[0], lo[1]);
            } else {
              *reinterpret_cast<uint4*>(s.q[x][0] + off) =
                  make_uint4(hi[0], hi[1], hi[2], hi[3]);
            }
          }
        }
        c = rsqrtf(float(DIM)) * kLog2e / c;
        fence_proxy_async();
        tc::fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&s.q_full[x]);
      }
      float m = -INFINITY, m_slot = -INFINITY;  // now; of what the slot holds
      float* po = a.chunk_part + size_t(g.slot) * 256 * DIM + (x * 128 + t) * 4;
      float2 sum0 = make_float2(0, 0), sum1 = sum0;
      for (int j = 0; j < g.count; ++j) {
        const int key0 = (g.lo_unit + g.u0 + j) * kChunkKeys;
        const bool flush = j % kFlushTiles<T> == 0;
        if (kCanFlush && flush && j > 0) {
          // while S_j is computed
          if (!wait_all(&s.o_full[x], o_uses++ & 1)) {
            ok = false;
            break;
          }
          tc::fence_after();
          // (no reader but this thread: the additions need no answer)
          const bool moved = __any_sync(0xffffffffu, !(m_slot == m));
          const bool first = j == kFlushTiles<T>;
          const float f = m_slot == -INFINITY ? 0.0F : ex2(m_slot - m);
#pragma unroll 1
          for (int i = 0; i < DIM / 32; ++i) {
            uint32_t ov[32];
            tc::ld32(to + i * 32, ov);
            tc::wait_ld();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              float4* at = reinterpret_cast<float4*>(po + (i * 8 + k) * 1024);
              float4 v = make_float4(__uint_as_float(ov[4 * k]),
                                     __uint_as_float(ov[4 * k + 1]),
                                     __uint_as_float(ov[4 * k + 2]),
                                     __uint_as_float(ov[4 * k + 3]));
              if (!first && !moved) {
                asm volatile(
                    "red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at),
                    "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                    : "memory");
                continue;
              }
              if (!first) {
                const float4 old = __ldcg(at);
                v = make_float4(fmaf(old.x, f, v.x), fmaf(old.y, f, v.y),
                                fmaf(old.z, f, v.z), fmaf(old.w, f, v.w));
              }
              __stcg(at, v);
            }
          }
          m_slot = m;
        }
        if (!wait_all(&s.s_full[x], (tiles + j) & 1)) {
          ok = false;
          break;
        }
        tc::fence_after();
        // S is read twice, for the maximum and for the probabilities: with
        // all 128 values and the packed P live, registers would spill
        const bool edge = range.edge(key0);
        const int hi = own - key0, lo = oldest - key0;
        // columns first .. first + 31 that the row does not see become -inf
        const auto mask = [&](uint32_t(&v)[32], int first) {
          if (!edge)
            return;
          const int a0 = max(lo - first, 0), a1 = min(hi - first, 31);
          const uint32_t seen =
              a1 < a0 || a0 > 31 ? 0u
                                 : (0xffffffffu >> (31 - (a1 - a0))) << a0;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(seen >> i & 1))
              v[i] = __float_as_uint(-INFINITY);
        };
        uint32_t v0[32], v1[32];
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const auto largest = [&](const uint32_t(&v)[32]) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tops[k] = max_nan(tops[k],
                                max_nan(__uint_as_float(v[i + k]),
                                        __uint_as_float(v[i + k + 4])));
        };
#pragma unroll 1
        for (int first = 64; first >= 0; first -= 64) {
          tc::ld32(ts + first, v0);
          tc::ld32(ts + first + 32, v1);
          tc::wait_ld();
          mask(v0, first);
          mask(v1, first + 32);
          largest(v0);
          largest(v1);
        }
        const float top =
            max_nan(max_nan(tops[0], tops[1]), max_nan(tops[2], tops[3])) * c;
        // (the difference is exact where it matters; m + kTopLimit may round)
        const bool move = !(top <= m) && !(top - m <= kTopLimit);
        if (__any_sync(0xffffffffu, move)) {
          float alpha = 1;
          if (move) {
            alpha = ex2(m - (top - kTopMoved));
            // a NaN or an infinite score makes the row NaN
            m = top < INFINITY ? top - kTopMoved : NAN;
            sum0 = make_float2(sum0.x * alpha, sum0.y * alpha);
            sum1 = make_float2(sum1.x * alpha, sum1.y * alpha);
          }
          // O follows the reference, unless it begins anew
          if (!flush) {
#pragma unroll 1
            for (int i = 0; i < DIM / 16; ++i) {
              uint32_t ov[16];
              tc::ld16(to + i * 16, ov);
              tc::wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k)
                ov[k] = __float_as_uint(__uint_as_float(ov[k]) * alpha);
              tc::st16(to + i * 16, ov);
            }
          }
        }
        const float shift = m == -INFINITY ? 0.0F : -m;
        const bool large = __any_sync(0xffffffffu, fabsf(shift) > kLargeScore);
        if (large) {  // columns 0 .. 63 are in v0 and v1, the others still in S
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            v0[i] = __float_as_uint(__fmul_rn(__uint_as_float(v0[i]), c));
            v1[i] = __float_as_uint(__fmul_rn(__uint_as_float(v1[i]), c));
          }
#pragma unroll 1
          for (int first = 64; first < 128; first += 16) {
            uint32_t v[16];
            tc::ld16(ts + first, v);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              v[i] = __float_as_uint(__fmul_rn(__uint_as_float(v[i]), c));
            tc::st16(ts + first, v);
          }
          tc::wait_st();
        }
        const float c_now = large ? 1.0F : c;
        const float2 c2 = make_float2(c_now, c_now);
        const float2 shift2 = make_float2(shift, shift);
        uint32_t ph[16], pl[16];
        const auto compute = [&](const uint32_t(&v)[32]) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 p = fma2(make_float2(__uint_as_float(v[2 * i]),
                                        __uint_as_float(v[2 * i + 1])),
                            c2, shift2);
            p.x = ex2(p.x);
            p.y = ex2(p.y);
            if (i % 2)
              sum1 = add2(sum1, p);
            else
              sum0 = add2(sum0, p);
            ph[i] = half2_bits(p.x, p.y);
            if constexpr (TERMS == 2) {
              const float2 back = bits_half2(ph[i]);
              pl[i] = half2_bits(p.x - back.x, p.y - back.y);
            } else {
              (void)pl;
            }
          }
        };
        // P over S: the fp16 terms of keys 32 i .. + 31 take the 32 columns
        // (16 a term) their scores were read from
        const auto store = [&](int first) {
          tc::st16(ts + first, ph);
          if constexpr (TERMS == 2)
            tc::st16(ts + first + 16, pl);
        };
        const auto arrive = [&](int third) {
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0)
            mbar_arrive(&s.p_full[x][third]);
        };
        // (v0 and v1 hold columns 0 .. 63; a piece is handed over once the
        // next one is worked out, so that its stores need no waiting for)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half) {
            tc::wait_ld();
            mask(v0, 64);
            tc::ld32(ts + 96, v1);
          }
          compute(v0);
          if (half)
            arrive(0);
          store(64 * half);
          if (half) {
            tc::wait_ld();
            mask(v1, 96);
          } else {
            tc::ld32(ts + 64, v0);
          }
          compute(v1);
          if (half)
            arrive(1);
          store(64 * half + 32);
        }
        arrive(2);
      }
      // ---- epilogue
      if (ok)
        ok = wait_all(&s.o_full[x], o_uses++ & 1);
      if (!ok)
        break;
      tc::fence_after();
      const int seg0 = (g.lo_unit + g.u0) * kChunkKeys;
      const float l = (sum0.x + sum1.x) + (sum0.y + sum1.y);
      // (every tile's clearing precedes its P V, which precedes o_full)
      const bool odd = *reinterpret_cast<volatile int*>(&s.odd_values) != 0;
      const bool whole = g.count == g.n_units;
      const bool flushed = kCanFlush && g.count > kFlushTiles<T>;
      const float f = m_slot == -INFINITY ? 0.0F : ex2(m_slot - m);
      float factor = 1;
      if (whole) {
        factor = l == 0 ? 0.0F : 1.0F / l;
        if (a.gate && live)
          factor /= 1 + expf(-to_float(static_cast<const T*>(
                            a.gate)[row * a.ldg + head]));
        if (a.lse && live)
          a.lse[row * a.heads + head] = (m + log2f(l)) * kLn2;
      } else {
        float2* pm = reinterpret_cast<float2*>(
            a.chunk_part + size_t(2 * kChunkCtas) * 256 * DIM);
        pm[g.slot * 256 + x * 128 + t] = make_float2(m, l);
      }
      // whole rows go through the warp's part of the Q buffer (16-byte piece
      // i of row r at i ^ (r & 7)), then out a row at a time
      uint8_t* stage = s.q[x][0] + (warp % 4) * 32 * DIM * sizeof(T);
      constexpr int kPieces = DIM * sizeof(T) / 16;
#pragma unroll
      for (int i = 0; i < DIM / 32; ++i) {
        uint32_t ov[32];
        tc::ld32(to + i * 32, ov);
        tc::wait_ld();
        if (flushed) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 old = __ldcg(
                reinterpret_cast<const float4*>(po + (i * 8 + k) * 1024));
            const float o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              ov[4 * k + e] = __float_as_uint(
                  fmaf(o[e], f, __uint_as_float(ov[4 * k + e])));
          }
        }
        if (odd && live)
          // values that were cleared although this row sees them
          for (int key = max(oldest, seg0);
               key <= min(own, seg0 + g.count * kChunkKeys - 1); ++key) {
            if (!range.edge(key / kChunkKeys * kChunkKeys))
              continue;  // not a tile that was cleared
            const int pool = paged_row(a.t, a.t.table, g.seq, key);
            if (pool < 0)
              continue;
            const __half* v =
                a.t.v + (size_t(pool) * kvh + g.h) * DIM + i * 32;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if ((__half_as_ushort(v[k]) & 0x7C00) == 0x7C00)
                ov[k] = __float_as_uint(__uint_as_float(ov[k]) +
                                        __half2float(v[k]));
          }
        if (!whole) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            *reinterpret_cast<uint4*>(po + (i * 8 + k) * 1024) =
                make_uint4(ov[4 * k], ov[4 * k + 1], ov[4 * k + 2],
                           ov[4 * k + 3]);
        } else {
#pragma unroll
          for (int k = 0; k < 32 / kVec; ++k) {
            alignas(16) T y[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e)
              y[e] = from_float<T>(__uint_as_float(ov[k * kVec + e]) * factor);
            const int piece = i * (32 / kVec) + k;
            *reinterpret_cast<uint4*>(
                stage + (lane * kPieces + (piece ^ (lane & 7))) * 16) =
                *reinterpret_cast<const uint4*>(y);
          }
        }
      }
      if (whole) {
        __syncwarp();
        const size_t offset = row * a.ldo + size_t(head) * DIM;
        const unsigned alive = __ballot_sync(0xffffffffu, live);
#pragma unroll 4
        for (int i = 0; i < 32; i += kRowsAtOnce) {
          const int r = i + sub;
          const size_t at =
              __shfl_sync(0xffffffffu, (unsigned long long)offset, r);
          if (alive >> r & 1)
            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at +
                                      part * kVec) =
                *reinterpret_cast<const uint4*>(
                    stage + (r * kPieces + (part ^ (r & 7))) * 16);
        }
      }
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&s.q_free[x]);
      tiles += g.count;
      ++segments;
    }
    // pairs of row tiles that see no key
    for (int j = blockIdx.x; j < a.t.sequences; j += gridDim.x) {
      const PagedSequence q = paged_sequence(a.t, j);
      const int pairs = q.length < q.n ? chunk_pairs(q, group) : 0;
      int lo;
      for (int p = 0; p < pairs; ++p) {
        if (chunk_units(q, group, a.window, p, lo))
          continue;
        for (int i = p * 2 * QB + warp; i < min(q.n, (p + 1) * 2 * QB);
             i += 8) {
          const size_t row = size_t(q.row0) + i;
          for (int e = lane; e < a.heads * DIM; e += 32)
            static_cast<T*>(a.out)[row * a.ldo + e] = from_float<T>(0);
          for (int e = lane; a.lse && e < a.heads; e += 32)
            a.lse[row * a.heads + e] = -INFINITY;
        }
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 9) {
    tc::fence_after();
    tc::dealloc(tmem, kColumns);
  }
}

template <typename T, int DIM>
cudaError_t launch(const PagedAttentionArgs& a, cudaStream_t stream) {
  const auto kernel = paged_chunk_kernel<T, DIM>;
  const int smem = int(sizeof(ChunkSmem<DIM, sizeof(T) == 4 ? 2 : 1>)) + 1024;
  if (cudaError_t e =
          ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem))
    return e;
  return launch_kernel(kernel, dim3(kChunkCtas), dim3(kThreads), smem, stream,
                       true, a);
}
template <typename T>
cudaError_t launch(const PagedAttentionArgs& a, int dim, cudaStream_t stream) {
  return dim == 64 ? launch<T, 64>(a, stream) : launch<T, 128>(a, stream);
}

}  // namespace

size_t paged_chunk_floats(int dim) {
  return size_t(2 * kChunkCtas) * 256 * (dim + 2) +
         kChunkCtas * sizeof(PagedRecord) / 4;
}

cudaError_t launch_paged_chunk(const PagedAttentionArgs& a, uint32_t type,
                               int dim, cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, dim, stream)
                            : launch<__nv_bfloat16>(a, dim, stream);
}

}  // namespace lfm3
