// Attention weight per cached key, accumulated (lfm3_cuda_paged_key_weights):
//
//   w_t += sum over new rows r and heads h of exp(q_rh k_t rsqrt(dim) - lse_rh)
//
// Three kernels. `terms` turns the queries into fp16 terms (two for FP32, as
// the attention kernels take them) with each row's power of two and lse beside
// them. `sums` computes S^T = K Q^T on the tcgen05 tensor cores with the keys
// as rows: a thread owns a key (its tensor-memory lane) and a row sum is an
// addition in a register, where the other way round it would be a sum over
// lanes. `update` adds what several blocks share of a key tile.
// `sums` works on pairs of 128-key tiles: the keys of a KV head stay in shared
// memory while its columns (query, head of the group) stream through in blocks
// of 128, and the warps 0-3 and 4-7 (a key tile each) read the scores from one
// half of tensor memory while the other half is computed. One exponential per
// (key, column) is the bound for chunks, reading K for single tokens (columns
// are then a multiple of 16). Blocks take equal shares of (key pair, KV head,
// column block) units (paged_plan.cuh); sums run in the order of units, then of
// blocks. Measured: 512 bf16 rows at depth 8192 (69 M exponentials, 15 us of
// the special function units) 43.6 us for the three kernels (`sums` waits for
// tensor memory: the special function units are busy for 44 %, issue slots for
// 24 % of it); 16 FP32 single tokens over 1024 to 8192 keys 19 us, K at 3.6
// TB/s. A polynomial on the FMA pipe for a quarter of the exponentials was no
// faster (45 us: the choice between the two costs what it saves), nor were 64
// columns a read (43.6 us).
// Warps: 8 TMA, 9 tensor memory and MMA, 10 the columns' factors, 11 segments.
#include <algorithm>
#include <type_traits>

#include "kernels.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "tcgen05.cuh"
#include "tensor_map.hpp"

namespace lfm3 {
namespace {

constexpr int kThreads = 12 * 32;
constexpr uint32_t kColumns = 512;
constexpr uint32_t kSlab = 128 * 128;  // bytes of [128 rows][64 dims]
constexpr int kPlanned = 4;            // segments worked out ahead
constexpr int kFewQueries = 4;         // copied one by one, not as a block

template <int DIM>
struct __align__(1024) WeightSmem {
  static constexpr int kSlabs = DIM / 64;
  static constexpr int kTile = kSlabs * kSlab;
  static constexpr int kKeyStages = 2;
  static constexpr int kTermStages = DIM == 128 ? 2 : 6;
  uint8_t k[kKeyStages][2][kTile];
  uint8_t q[kTermStages][kTile];
  float4 factors[2][64];  // of two columns: c, c', -lse, -lse'
  uint32_t without[2][5];  // columns whose lse is infinite, and whether any is
  uint64_t k_full[kKeyStages], k_empty[kKeyStages];
  uint64_t q_full[kTermStages], q_empty[kTermStages];
  uint64_t f_full[2], f_empty[2];
  uint64_t d_full[2][2], d_empty[2][2];  // [half of tensor memory][key tile]
  uint64_t idle;
  uint64_t seg_full[kPlanned], seg_empty[kPlanned];
  WeightSegment seg[kPlanned];
  uint32_t tmem;
};

// ---- terms: a warp per (row, head)
template <typename T, int DIM>
__global__ void __launch_bounds__(256)
    paged_terms_kernel(const __grid_constant__ PagedKeyWeightsArgs a) {
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  constexpr int kPer = DIM / 32;
  const int lane = threadIdx.x % 32;
  grid_dependency_wait();
  allow_dependents();
  const int64_t items = int64_t(a.t.rows) * a.heads;
  for (int64_t i = int64_t(blockIdx.x) * 8 + threadIdx.x / 32; i < items;
       i += int64_t(gridDim.x) * 8) {
    const int64_t r = i / a.heads, h = i - r * a.heads;
    const T* src = static_cast<const T*>(a.q) + size_t(r) * a.ldq +
                   size_t(h) * DIM + lane * kPer;
    float x[kPer], top = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      x[e] = to_float(src[e]);
      top = fmaxf(top, fabsf(x[e]));
    }
    const float scale = row_scale(warp_max(top));
    alignas(8) __half hi[kPer], lo[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const SplitPair t = split_value(x[e] * scale);
      hi[e] = t.hi;
      lo[e] = t.lo;
    }
    __half* dst = a.terms + size_t(i) * DIM + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; e += 2) {
      *reinterpret_cast<__half2*>(dst + e) = __halves2half2(hi[e], hi[e + 1]);
      if constexpr (TERMS == 2)
        *reinterpret_cast<__half2*>(dst + size_t(items) * DIM + e) =
            __halves2half2(lo[e], lo[e + 1]);
    }
    if (lane == 0) {
      // a row without keys (lse -inf) adds nothing
      const float lse = a.lse[i];
      a.factors[i] = lse == -INFINITY
                         ? make_float2(0, INFINITY)
                         : make_float2(rsqrtf(float(DIM)) * kLog2e / scale,
                                       lse * kLog2e);
    }
  }
}

// The sum that key `key` of a sequence gained goes to its place.
__device__ __forceinline__ void add_weight(const PagedKeyWeightsArgs& a,
                                           const PagedSequence& q, int seq,
                                           int key, float sum) {
  if (key >= q.length)
    return;
  const int pool = paged_row(a.t, a.t.table, seq, key);
  if (pool < 0) {
    report_error(kErrPagedTable);
    return;
  }
  // rows new in this batch start from 0
  a.weights[pool] = key >= q.length - q.n ? sum : a.weights[pool] + sum;
}

// A shared key pair's record: its slots, and its place.
struct WeightRecord {
  int parts, slot, seq, pair;
};
// Bytes of the slots of sums and the records behind them, and of the factors:
// every part of the workspace begins on a 256-byte boundary.
constexpr size_t kPartBytes =
    (size_t(2 * kWeightCtas) * kWeightKeys * sizeof(float) +
     kWeightCtas * sizeof(WeightRecord) + 255) / 256 * 256;
constexpr size_t factor_bytes(size_t values) {
  return (values * sizeof(float2) + 255) / 256 * 256;
}

template <int DIM, int TERMS>
__global__ void __launch_bounds__(kThreads, 1)
    paged_sums_kernel(const __grid_constant__ PagedKeyWeightsArgs a) {
  using Smem = WeightSmem<DIM>;
  constexpr int kSlabs = Smem::kSlabs;
  constexpr int kKeyStages = Smem::kKeyStages;
  constexpr int kTermStages = Smem::kTermStages;
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int kvh = a.t.kv_heads, group = a.heads / kvh;
  const int QB = chunk_queries(group);  // queries of a column block
  if (tid == 0) {
    for (int i = 0; i < kKeyStages; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
    }
    for (int i = 0; i < kTermStages; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.f_full[i], 1);
      mbar_init(&s.f_empty[i], 8);
      for (int x = 0; x < 2; ++x) {
        mbar_init(&s.d_full[i][x], 1);
        mbar_init(&s.d_empty[i][x], 4);
      }
    }
    for (int i = 0; i < kPlanned; ++i) {
      mbar_init(&s.seg_full[i], 1);
      mbar_init(&s.seg_empty[i], 11);  // every other warp
    }
    mbar_init(&s.idle, 1);
    fence_barrier_init();
    prefetch_map(&a.kmap);
    for (int t = 0; t < TERMS; ++t) {
      prefetch_map(&a.qmap[t]);
      prefetch_map(&a.qmap1[t]);
    }
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
  WeightSegment g;
  uint32_t planned = 0;
  // a warp's lanes give up together
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) ||
           __all_sync(0xffffffffu, mbar_wait(bar, parity, kErrPagedWait));
  };
  // The next segment (warp-wide): false at the end of the block's share.
  const auto next_segment = [&]() {
    const uint32_t i = planned % kPlanned;
    ok = ok && wait(&s.seg_full[i], (planned / kPlanned) & 1);
    if (!ok)
      return false;
    g = s.seg[i];
    __syncwarp();
    if (lane == 0)
      mbar_arrive(&s.seg_empty[i]);
    ++planned;
    return g.count > 0;
  };
  // queries of column block b, and columns of the MMAs
  const auto queries = [&](int b) { return min(QB, g.q.n - b * QB); };

  if (warp == 11) {
    // ---- the block's segments, then one with count 0
    PagedLine line(a.t, WeightUnits{group, a.window});
    if (line.broken && blockIdx.x == 0)
      report_error(kErrPagedTable);
    const int64_t total = line.total * kvh;
    const int64_t share = paged_share(total, kWeightCtas, 1);
    const int64_t begin = share * blockIdx.x, end = min(begin + share, total);
    WeightRecord record{0, 0, 0, 0};
    int64_t at = begin;
    for (bool more = true; more && ok; ++planned) {
      more = weight_segment(line, group, a.window, at, end, g);
      if (!more)
        g.count = 0;
      g.slot = 2 * blockIdx.x + (at > begin ? 1 : 0);
      const uint32_t i = planned % kPlanned;
      if (planned >= kPlanned)
        ok = wait(&s.seg_empty[i], ((planned / kPlanned) - 1) & 1);
      if (lane == 0 && ok) {
        s.seg[i] = g;
        mbar_arrive(&s.seg_full[i]);
      }
      __syncwarp();
      if (more && g.count < g.n_units && g.u0 == 0)
        record = {paged_record(at, share, g.slot, g.n_units, g.q, 0, 0).parts,
                  g.slot, g.seq, g.pair};
      at += g.count;
    }
    if (lane == 0)
      reinterpret_cast<WeightRecord*>(
          a.part + size_t(2 * kWeightCtas) * kWeightKeys)[blockIdx.x] = record;
  } else if (warp == 8) {
    // ---- TMA: a KV head's keys once, then its column blocks' terms
    const int per = 128 / a.box_rows;  // boxes of a slab
    uint32_t keys = 0, terms = 0;
    while (next_segment()) {
      // the lane's part of a key pair
      const int key0 = g.pair * kWeightKeys;
      const int box = lane / kSlabs, slab = lane % kSlabs;
      const int boxes = min(2 * per, (g.q.length - key0 + a.box_rows - 1) /
                                         a.box_rows);
      int row = box < boxes ? paged_row(a.t, a.t.table, g.seq,
                                        key0 + box * a.box_rows)
                            : 0;
      if (row < 0) {
        report_error(kErrPagedTable);
        row = 0;
      }
      int h = -1;
      for (int u = g.u0; u < g.u0 + g.count && ok; ++u) {
        if (u / g.blocks != h) {
          h = u / g.blocks;
          const int st = keys % kKeyStages;
          if (keys >= kKeyStages)
            ok = wait(&s.k_empty[st], ((keys / kKeyStages) - 1) & 1);
          if (!ok)
            break;
          if (lane == 0)
            mbar_arrive_expect_tx(&s.k_full[st],
                                  uint32_t(boxes * kSlabs * a.box_rows) * 128);
          __syncwarp();
          if (box < boxes)
            tma_load_3d(s.k[st][box / per] + slab * kSlab +
                            box % per * a.box_rows * 128,
                        &a.kmap, 0, row, h * kSlabs + slab, &s.k_full[st]);
          ++keys;
        }
        const int b = g.lo + u - h * g.blocks, nq = queries(b);
        const bool few = nq <= kFewQueries;
        const int copies = kSlabs * (few ? nq : 1);
#pragma unroll
        for (int t = 0; t < TERMS; ++t, ++terms) {
          const int st = terms % kTermStages;
          if (terms >= kTermStages)
            ok = ok && wait(&s.q_empty[st], ((terms / kTermStages) - 1) & 1);
          if (!ok)
            break;
          // (a block's copy is whole: rows past the tensor land as zeros)
          if (lane == 0)
            mbar_arrive_expect_tx(
                &s.q_full[st],
                uint32_t(kSlabs * (few ? nq : QB) * group) * 128);
          __syncwarp();
          if (lane < copies)
            tma_load_5d(s.q[st] + lane % kSlabs * kSlab +
                            lane / kSlabs * group * 128,
                        few ? &a.qmap1[t] : &a.qmap[t], 0, 0,
                        g.q.row0 + b * QB + lane / kSlabs, lane % kSlabs, h,
                        &s.q_full[st]);
        }
      }
    }
    // no copy may still be landing when the block exits
    for (uint32_t i = keys > kKeyStages ? keys - kKeyStages : 0; i < keys; ++i)
      mbar_wait(&s.k_full[i % kKeyStages], (i / kKeyStages) & 1,
                kErrPagedWait);
    for (uint32_t i = terms > kTermStages ? terms - kTermStages : 0; i < terms;
         ++i)
      mbar_wait(&s.q_full[i % kTermStages], (i / kTermStages) & 1,
                kErrPagedWait);
  } else if (warp == 10) {
    // ---- the columns' factors, a unit ahead of the sums
    uint32_t done = 0;
    while (next_segment())
      for (int u = g.u0; u < g.u0 + g.count && ok; ++u, ++done) {
        const int h = u / g.blocks, b = g.lo + u - h * g.blocks;
        const int columns = queries(b) * group;
        float2 f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = lane * 4 + i;
          f[i] = make_float2(0, 0);
          if (col < columns)
            f[i] = a.factors[(size_t(g.q.row0) + b * QB + col / group) *
                                 a.heads +
                             h * group + col % group];
        }
        const int st = done % 2;
        if (done >= 2)
          ok = wait(&s.f_empty[st], ((done / 2) - 1) & 1);
        if (!ok)
          break;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          s.factors[st][lane * 2 + i] =
              make_float4(f[2 * i].x, f[2 * i + 1].x, -f[2 * i].y,
                          -f[2 * i + 1].y);
        uint32_t without = 0;  // a lane four columns, eight lanes a word
#pragma unroll
        for (int i = 0; i < 4; ++i)
          without |= uint32_t(f[i].y == INFINITY) << (lane % 8 * 4 + i);
        const bool any = __any_sync(0xffffffffu, without);
        if (any)
#pragma unroll
          for (int o = 1; o < 8; o <<= 1)
            without |= __shfl_xor_sync(0xffffffffu, without, o);
        if (lane % 8 == 0)
          s.without[st][lane / 8] = without;
        if (lane == 0)
          s.without[st][4] = any;
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&s.f_full[st]);
      }
  } else if (warp == 9) {
    // ---- every MMA, issued by one lane
    const bool lead = tc::elect();
    const auto uniform = [](int v) {
      return int(__reduce_max_sync(0xffffffffu, unsigned(v)));
    };
    const uint32_t tm = uniform(tmem);
    const uint64_t kdesc = tc::sw128_desc(s.k[0][0]);
    const uint64_t qdesc = tc::sw128_desc(s.q[0]);
    constexpr uint32_t kStep = Smem::kTile / 16;
    uint32_t keys = 0, terms = 0, done = 0;
    while (next_segment()) {
      const int blocks = uniform(g.blocks), u0 = uniform(g.u0);
      const int count = uniform(g.count);
      int h = -1;
      for (int i = 0; i < count && ok; ++i, ++done) {
        const int u = u0 + i;
        if (u / blocks != h) {
          h = u / blocks;
          ok = wait(&s.k_full[keys % kKeyStages], (keys / kKeyStages) & 1);
          ++keys;
        }
        const bool last_of_keys = i + 1 == count || (u + 1) / blocks != h;
        const int columns = queries(g.lo + u - h * blocks) * group;
        const uint32_t idesc =
            tc::f16_idesc(128, 16) +
            (uint32_t(uniform((columns + 15) / 16) - 1) << 18);
        const uint32_t half = done % 2;
        ok = ok &&
             (done < 2 || (wait(&s.d_empty[half][0], ((done / 2) - 1) & 1) &&
                           wait(&s.d_empty[half][1], ((done / 2) - 1) & 1)));
        if (!ok)
          break;
        const uint64_t k = kdesc + (keys - 1) % kKeyStages * 2 * kStep;
#pragma unroll
        for (int t = 0; t < TERMS; ++t, ++terms) {
          const uint32_t st = terms % kTermStages;
          ok = ok && wait(&s.q_full[st], (terms / kTermStages) & 1);
          if (!ok)
            break;
          tc::fence_after();
          const uint64_t q = qdesc + st * kStep;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int k16 = 0; k16 < DIM / 16; ++k16) {
              const int at = (k16 / 4) * (kSlab / 16) + (k16 % 4) * 2;
              tc::mma_lead(tm + (half * 2 + x) * 128, k + x * kStep + at,
                           q + at, idesc, t > 0 || k16 > 0, lead);
            }
            if (t == TERMS - 1)
              tc::commit_lead(&s.d_full[half][x], lead);
          }
          tc::commit_lead(&s.q_empty[st], lead);
        }
        if (last_of_keys)
          tc::commit_lead(&s.k_empty[(keys - 1) % kKeyStages], lead);
      }
    }
    tc::commit_lead(&s.idle, lead);
    mbar_wait(&s.idle, 0, kErrPagedWait);
  } else {
    // ---- the sums of key tile x: thread t owns key t
    const int x = warp / 4, t = tid % 128;
    const uint32_t lane_base = uint32_t((warp % 4) * 32) << 16;
    uint32_t done = 0;
    while (next_segment()) {
      const int key = g.pair * kWeightKeys + x * 128 + t;
      const int base = g.q.length - g.q.n;
      const int tile0 = g.pair * kWeightKeys + x * 128, tile1 = tile0 + 127;
      float2 sum0 = make_float2(0, 0), sum1 = sum0;
      for (int u = g.u0; u < g.u0 + g.count; ++u, ++done) {
        const int b = g.lo + u % g.blocks, nq = queries(b);
        const int columns = nq * group;
        const uint32_t half = done % 2;
        const uint32_t td = tmem + lane_base + (half * 2 + x) * 128;
        ok = ok && wait(&s.f_full[half], (done / 2) & 1) &&
             wait(&s.d_full[half][x], (done / 2) & 1);
        if (!ok)
          break;
        tc::fence_after();
        // Queries q0 .. q0 + nq - 1 of the block; every one sees every key of
        // the tile unless this is an edge. A key is seen from query
        // key - base on, and by `window` of them. Queries without lse are left
        // out the same way: 2^(x - inf) would be NaN for scores that are.
        const int q0 = b * QB;
        const bool edge = tile1 > base + q0 ||
                          (a.window > 0 &&
                           tile0 <= base + q0 + nq - 1 - a.window) ||
                          columns % 32 != 0 || s.without[half][4];
        const int64_t query = int64_t(key) - base - q0;
        // the key's columns: first .. last - 1
        const int first = int(min(max(query, int64_t(0)), int64_t(nq))) * group;
        const int last =
            a.window > 0
                ? int(min(max(query + a.window, int64_t(0)), int64_t(nq))) *
                      group
                : columns;
        const auto add_up = [&](auto some_hidden) {
#pragma unroll 1
          for (int c0 = 0; c0 < columns; c0 += 32) {
            uint32_t v[32];
            tc::ld32(td + c0, v);
            float4 f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              f[i] = s.factors[half][c0 / 2 + i];
            uint32_t seen = 0xffffffffu;
            if constexpr (some_hidden) {
              // columns a0 .. a1 - 1 of the 32 see the key
              const unsigned a0 = max(first - c0, 0), a1 = max(last - c0, 0);
              seen = a1 <= a0 || a0 > 31
                         ? 0u
                         : (0xffffffffu >> (32 - (min(a1, 32u) - a0))) << a0;
              seen &= ~s.without[half][c0 / 32];
            }
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2 p = fma2(make_float2(__uint_as_float(v[2 * i]),
                                          __uint_as_float(v[2 * i + 1])),
                              make_float2(f[i].x, f[i].y),
                              make_float2(f[i].z, f[i].w));
              if constexpr (some_hidden) {
                if (!(seen >> (2 * i) & 1))
                  p.x = -INFINITY;
                if (!(seen >> (2 * i + 1) & 1))
                  p.y = -INFINITY;
              }
              p.x = ex2(p.x);
              p.y = ex2(p.y);
              if (i % 2)
                sum1 = add2(sum1, p);
              else
                sum0 = add2(sum0, p);
            }
          }
        };
        if (edge)
          add_up(std::true_type{});
        else
          add_up(std::false_type{});
        tc::fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s.d_empty[half][x]);
          mbar_arrive(&s.f_empty[half]);
        }
      }
      if (!ok)
        break;
      const float sum = (sum0.x + sum0.y) + (sum1.x + sum1.y);
      if (g.count == g.n_units)
        add_weight(a, g.q, g.seq, key, sum);
      else
        a.part[size_t(g.slot) * kWeightKeys + x * 128 + t] = sum;
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 9) {
    tc::fence_after();
    tc::dealloc(tmem, kColumns);
  }
}

// ---- update: block = record, thread = key
__global__ void __launch_bounds__(kWeightKeys)
    paged_update_kernel(const __grid_constant__ PagedKeyWeightsArgs a) {
  allow_dependents();
  grid_dependency_wait();
  const WeightRecord r = reinterpret_cast<const WeightRecord*>(
      a.part + size_t(2 * kWeightCtas) * kWeightKeys)[blockIdx.x];
  if (r.parts == 0)
    return;
  const PagedRecord slots{r.parts, r.slot, 0, 0, 0, 0};
  float sum = 0;
  for (int p = 0; p < r.parts; ++p)
    sum += a.part[size_t(record_slot(slots, p)) * kWeightKeys + threadIdx.x];
  add_weight(a, paged_sequence(a.t, r.seq), r.seq,
             r.pair * kWeightKeys + threadIdx.x, sum);
}

template <typename T, int DIM>
cudaError_t launch(PagedKeyWeightsArgs a, cudaStream_t stream) {
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  const int kvh = a.t.kv_heads, group = a.heads / kvh;
  const size_t values = size_t(a.t.rows) * a.heads;
  char* space = static_cast<char*>(a.workspace);
  a.part = reinterpret_cast<float*>(space);
  a.factors = reinterpret_cast<float2*>(space + kPartBytes);
  a.terms =
      reinterpret_cast<__half*>(space + kPartBytes + factor_bytes(values));
  a.box_rows = std::min(a.t.page_rows & -a.t.page_rows, 128);
  cudaError_t e;
  if ((e = encode_pool_map(&a.kmap, a.t.k, a.t.pages * a.t.page_rows, kvh, DIM,
                           a.box_rows, 1)))
    return e;
  for (int t = 0; t < TERMS; ++t) {
    const __half* terms = a.terms + t * values * DIM;
    if ((e = encode_group_map(&a.qmap1[t], terms, a.t.rows, kvh, group, DIM,
                              1)) ||
        (e = encode_group_map(&a.qmap[t], terms, a.t.rows, kvh, group, DIM,
                              chunk_queries(group))))
      return e;
  }
  const int64_t blocks = std::min<int64_t>((int64_t(values) + 7) / 8, 148 * 8);
  if ((e = launch_kernel(paged_terms_kernel<T, DIM>, dim3(unsigned(blocks)),
                         dim3(256), 0, stream, true, a)))
    return e;
  const auto kernel = paged_sums_kernel<DIM, TERMS>;
  const int smem = int(sizeof(WeightSmem<DIM>)) + 1024;
  if ((e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) ||
      (e = launch_kernel(kernel, dim3(kWeightCtas), dim3(kThreads), smem,
                         stream, true, a)))
    return e;
  return launch_kernel(paged_update_kernel, dim3(kWeightCtas),
                       dim3(kWeightKeys), 0, stream, true, a);
}
template <typename T>
cudaError_t launch(const PagedKeyWeightsArgs& a, int dim,
                   cudaStream_t stream) {
  return dim == 64 ? launch<T, 64>(a, stream) : launch<T, 128>(a, stream);
}

}  // namespace

size_t paged_key_weights_workspace(const PagedTables& t, int dim, int heads) {
  const size_t values = size_t(t.rows) * heads;
  return kPartBytes + factor_bytes(values) + values * dim * 2 * sizeof(__half);
}

cudaError_t launch_paged_key_weights(const PagedKeyWeightsArgs& a,
                                     uint32_t type, int dim,
                                     cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, dim, stream)
                            : launch<__nv_bfloat16>(a, dim, stream);
}

}  // namespace lfm3
