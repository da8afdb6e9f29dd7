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
// FP32 queries are two fp16 terms (two MMAs for S, both terms of P fill the
// 128 columns of S, two MMAs for O): 22 bits where a 16-bit type has one term.
// Rows are scaled to fp16's range by a power of two first.
// A row's probabilities are 2^(x - m) with a reference m that trails the
// running maximum: 2^7 for the maximum when m moves, 2^15 at most before it
// moves again, so it (and with it O in tensor memory) moves rarely and
// small probabilities stay clear of fp16's subnormals.
// Masked keys. A key that a row does not see has probability 0, but 0 times a
// NaN or an infinity in V would still reach the row's sums. In tiles where
// some row sees less than all keys (the diagonal, a window's edge, the last
// page's tail) the softmax warps therefore clear rows that no row of the pair
// sees and values that are not finite before P V runs; rows that do see such a
// value get it added at the end.
// Blocks take equal shares of the batch's (row tile pair, KV head, key tile)
// units (paged_plan.cuh), so one long history is split over all SMs. Warps:
// 0-3 and 4-7 softmax and epilogue, 8 TMA, 9 tensor memory and (one thread)
// every MMA. Every wait is bounded.
#include "kernels.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "tcgen05.cuh"
#include "tensor_map.hpp"

namespace lfm3 {
namespace {

constexpr int kThreads = 10 * 32;
constexpr uint32_t kColS = 128, kColO = 256, kColumns = 512;
constexpr uint32_t kSlab = 128 * 128;  // bytes of [128 rows][64 dims]
// exponents (base 2) of a row's largest probability: when the reference
// moves, and when it has to move again
constexpr float kTopMoved = 7.0F, kTopLimit = 15.0F;

template <int DIM, int TERMS>
struct __align__(1024) ChunkSmem {
  static constexpr int kSlabs = DIM / 64;
  static constexpr int kTile = kSlabs * kSlab;
  static constexpr int kStages =
      DIM == 128 ? (TERMS == 2 ? 3 : 5) : (TERMS == 2 ? 8 : 10);
  uint8_t q[2][TERMS][kTile];
  uint8_t kv[kStages][kTile];  // K_0 V_0 K_1 V_1 ... in turn
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], idle;
  uint32_t tmem;
  int odd_values;  // a value that is not finite was cleared in this segment
};

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 bits_half2(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
// Whether one of a word's two fp16 values is infinite or NaN.
__device__ __forceinline__ bool not_finite2(uint32_t u) {
  return (((u & 0x7C007C00u) + 0x04000400u) & 0x80008000u) != 0;
}

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
      mbar_init(&s.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 4);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);
      mbar_init(&s.o_full[i], 1);
    }
    mbar_init(&s.idle, 1);
    s.odd_values = 0;
    fence_barrier_init();
  }
  if (warp == 9)
    tc::alloc(&s.tmem, kColumns);
  if (tid == 0) {
    prefetch_map(&a.kmap);
    prefetch_map(&a.vmap);
  }
  if (!a.behind_decode)
    grid_dependency_wait();
  allow_dependents();
  const auto units = [&](const PagedSequence& q) {
    return chunk_sequence_units(q, group, a.window);
  };
  const PagedLine line(a.t, units);
  if (line.broken && blockIdx.x == 0 && warp == 0)
    report_error(kErrPagedTable);
  const int64_t total = line.total * kvh;
  const int64_t share = paged_share(total, gridDim.x, kChunkMinUnits);
  const int64_t begin = share * blockIdx.x, end = min(begin + share, total);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = s.tmem;
  bool ok = true;
  ChunkSegment g;
  // A barrier's phase is the parity of its completed uses: loads so far, and
  // per row tile the key tiles and segments so far in which it took part.

  if (warp == 8) {
    // ---- TMA: K and V tiles, a lane per box
    const int per = 128 / a.box_rows;  // boxes of a slab
    uint32_t loads = 0;
    for (int64_t at = begin;
         ok && chunk_segment(line, group, a.window, at, end, g); at += g.count)
      for (int i = 0; i < 2 * g.count && ok; ++i, ++loads) {
        const int st = loads % kStages;
        if (loads >= kStages)
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&s.kv_empty[st],
                                    ((loads / kStages) - 1) & 1,
                                    kErrPagedWait));
        if (!ok)
          break;
        const int key0 = (g.lo_unit + g.u0 + i / 2) * kChunkKeys;
        // boxes that hold rows of the sequence
        const int boxes =
            min(per, (g.q.length - key0 + a.box_rows - 1) / a.box_rows);
        if (lane == 0)
          mbar_arrive_expect_tx(&s.kv_full[st],
                                uint32_t(boxes * kSlabs * a.box_rows) * 128);
        __syncwarp();
        for (int b = lane; b < boxes * kSlabs; b += 32) {
          const int box = b / kSlabs, slab = b % kSlabs;
          int row = paged_row(a.t, a.t.table, g.seq, key0 + box * a.box_rows);
          if (row < 0) {
            report_error(kErrPagedTable);
            row = 0;
          }
          tma_load_3d(s.kv[st] + slab * kSlab + box * a.box_rows * 128,
                      i % 2 ? &a.vmap : &a.kmap, 0, row, g.h * kSlabs + slab,
                      &s.kv_full[st]);
        }
      }
    // no copy may still be landing when the block exits
    for (uint32_t i = loads > kStages ? loads - kStages : 0; i < loads; ++i)
      mbar_wait(&s.kv_full[i % kStages], (i / kStages) & 1, kErrPagedWait);
  } else if (warp == 9) {
    // ---- every MMA, one thread
    uint32_t loads = 0, tiles[2] = {0, 0}, segments[2] = {0, 0};
    for (int64_t at = begin;
         ok && chunk_segment(line, group, a.window, at, end, g);
         at += g.count, loads += 2 * g.count) {
      const int two = g.q.n - g.pair * 2 * QB > QB;  // row tile 1 is there
      if (lane == 0) {
        const auto full = [&](int i) {  // load i of this segment has landed
          const uint32_t l = loads + i;
          return mbar_wait(&s.kv_full[l % kStages], (l / kStages) & 1,
                           kErrPagedWait);
        };
        const auto release = [&](int i) {
          tc::commit(&s.kv_empty[(loads + i) % kStages]);
        };
        const auto scores = [&](int x, int j) {
          const uint8_t* k = s.kv[(loads + 2 * j) % kStages];
#pragma unroll
          for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int k16 = 0; k16 < DIM / 16; ++k16)
              tc::mma(tmem + x * kColS,
                      tc::sw128_desc(s.q[x][t] + (k16 / 4) * kSlab) +
                          (k16 % 4) * 2,
                      tc::sw128_desc(k + (k16 / 4) * kSlab) + (k16 % 4) * 2,
                      kIdescS, t > 0 || k16 > 0);
          tc::commit(&s.s_full[x]);
        };
        const auto values = [&](int x, int j) {
          const uint64_t v =
              tc::sw128_mn_desc(s.kv[(loads + 2 * j + 1) % kStages], kSlab);
#pragma unroll
          for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int k16 = 0; k16 < 8; ++k16)
              tc::mma_ts(tmem + kColO + x * 128,
                         tmem + x * kColS + t * 64 + k16 * 8, v + k16 * 128,
                         kIdescO, j > 0 || t > 0 || k16 > 0);
        };
        ok = mbar_wait(&s.q_full[0], segments[0] & 1, kErrPagedWait) && full(0);
        if (ok) {
          tc::fence_after();
          scores(0, 0);
          if (two) {
            ok = mbar_wait(&s.q_full[1], segments[1] & 1, kErrPagedWait);
            tc::fence_after();
            if (ok)
              scores(1, 0);
          }
          release(0);
        }
        for (int j = 0; j < g.count && ok; ++j) {
          const bool more = j + 1 < g.count;
          ok = full(2 * j + 1);
          for (int x = 0; x < 1 + two && ok; ++x) {
            ok = mbar_wait(&s.p_full[x], (tiles[x] + j) & 1, kErrPagedWait);
            if (!ok)
              break;
            tc::fence_after();
            values(x, j);
            if (x == two)
              release(2 * j + 1);
            if (more) {
              if (x == 0)
                ok = full(2 * j + 2);
              if (ok)
                scores(x, j + 1);
              if (x == two)
                release(2 * j + 2);
            } else {
              tc::commit(&s.o_full[x]);
            }
          }
        }
        for (int x = 0; x < 1 + two; ++x) {
          tiles[x] += g.count;
          ++segments[x];
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (lane == 0) {
      tc::commit(&s.idle);
      mbar_wait(&s.idle, 0, kErrPagedWait);
    }
  } else {
    // ---- softmax and epilogue of row tile x: thread t owns row t
    const int x = warp / 4, t = tid % 128;
    const uint32_t lane_base = uint32_t((warp % 4) * 32) << 16;
    const uint32_t ts = tmem + lane_base + x * kColS;
    const uint32_t to = tmem + lane_base + kColO + x * 128;
    // a warp's lanes give up together: tensor-memory accesses are warp-wide
    const auto wait_all = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, kErrPagedWait));
    };
    uint32_t loads = 0, tiles = 0, segments = 0;
    PagedRecord record{0, 0, 0, 0, 0, 0};
    for (int64_t at = begin;
         ok && chunk_segment(line, group, a.window, at, end, g);
         at += g.count, loads += 2 * g.count) {
      const int q0 = g.pair * 2 * QB;
      const int qlast = min(g.q.n, q0 + 2 * QB) - 1;
      const int base = g.q.length - g.q.n;
      if (x == 1 && g.q.n - q0 <= QB)
        continue;
      const int qi = q0 + x * QB + t / group, head = g.h * group + t % group;
      const bool live = t < QB * group && qi < g.q.n;
      const size_t row = size_t(g.q.row0) + (live ? qi : 0);
      // the row sees keys own - window + 1 .. own
      const int own = live ? base + qi : -1;
      const int oldest = a.window > 0 ? max(0, own - a.window + 1) : 0;
      // ... of which every row of the pair sees all_lo .. all_hi, some row
      // any_lo .. any_hi
      const int all_hi = base + q0, any_hi = base + qlast;
      const int all_lo =
          a.window > 0 ? max(0, base + qlast - a.window + 1) : 0;
      const int any_lo = a.window > 0 ? max(0, base + q0 - a.window + 1) : 0;
      float c;
      {
        // ---- Q row as fp16 terms
        const T* src = static_cast<const T*>(a.q) + row * a.ldq +
                       size_t(live ? head : 0) * DIM;
        constexpr int kVec = 16 / sizeof(T);
        uint4 raw[DIM / kVec];
        float top = 0;
#pragma unroll
        for (int i = 0; i < DIM / kVec; ++i) {
          raw[i] = live ? reinterpret_cast<const uint4*>(src)[i]
                        : make_uint4(0, 0, 0, 0);
          const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
          for (int k = 0; k < kVec; ++k)
            top = fmaxf(top, fabsf(to_float(e[k])));
        }
        const float scale = row_scale(top);
        c = rsqrtf(float(DIM)) * kLog2e / scale;
#pragma unroll
        for (int piece = 0; piece < DIM / 8; ++piece) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int e = piece * 8 + 2 * k;
            const T* p = reinterpret_cast<const T*>(raw) + e;
            const float v0 = to_float(p[0]) * scale, v1 = to_float(p[1]) * scale;
            hi[k] = half2_bits(v0, v1);
            const float2 back = bits_half2(hi[k]);
            lo[k] = half2_bits(v0 - back.x, v1 - back.y);
          }
          const uint32_t off =
              (piece / 8) * kSlab + tc::sw128_offset(t, piece % 8);
          *reinterpret_cast<uint4*>(s.q[x][0] + off) =
              make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if constexpr (TERMS == 2)
            *reinterpret_cast<uint4*>(s.q[x][TERMS - 1] + off) =
                make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async();
        tc::fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&s.q_full[x]);
      }
      float m = -INFINITY, l = 0;
      for (int j = 0; j < g.count; ++j) {
        const int key0 = (g.lo_unit + g.u0 + j) * kChunkKeys;
        if (!wait_all(&s.s_full[x], (tiles + j) & 1)) {
          ok = false;
          break;
        }
        tc::fence_after();
        uint32_t sv[128];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tc::ld32(ts + i * 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32 * i));
        tc::wait_ld();
        const bool edge = key0 + kChunkKeys - 1 > all_hi || key0 < all_lo;
        if (edge) {
          const int hi = own - key0, lo = oldest - key0;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i > hi || i < lo)
              sv[i] = __float_as_uint(-INFINITY);
          // clear what masked rows must not meet in V
          const uint32_t ld = loads + 2 * j + 1;
          if (!wait_all(&s.kv_full[ld % kStages], (ld / kStages) & 1)) {
            ok = false;
            break;
          }
          uint8_t* v = s.kv[ld % kStages];
          for (int i = t; i < 128 * kSlabs * 8; i += 128) {
            const int key = i / (8 * kSlabs), piece = i % (8 * kSlabs);
            uint4* at16 = reinterpret_cast<uint4*>(
                v + (piece / 8) * kSlab + tc::sw128_offset(key, piece % 8));
            if (key0 + key < any_lo || key0 + key > any_hi) {
              *at16 = make_uint4(0, 0, 0, 0);
              continue;
            }
            uint4 w = *at16;
            if (not_finite2(w.x) || not_finite2(w.y) || not_finite2(w.z) ||
                not_finite2(w.w)) {
              __half* e = reinterpret_cast<__half*>(&w);
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if ((__half_as_ushort(e[k]) & 0x7C00) == 0x7C00)
                  e[k] = __ushort_as_half(0);
              // (the flag first: the other row tile may find zeros here)
              *reinterpret_cast<volatile int*>(&s.odd_values) = 1;
              __threadfence_block();
              *at16 = w;
            }
          }
          fence_proxy_async();
        }
        float tops[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tops[i] = __uint_as_float(sv[i]);
#pragma unroll
        for (int i = 4; i < 128; ++i)
          tops[i % 4] = fmaxf(tops[i % 4], __uint_as_float(sv[i]));
        const float top =
            fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * c;
        const bool move = top > m + kTopLimit;
        float alpha = 1;
        if (move) {
          alpha = ex2(m - (top - kTopMoved));
          m = top - kTopMoved;
          l *= alpha;
        }
        const float shift = m == -INFINITY ? 0.0F : -m;
        uint32_t ph[64], pl[TERMS == 2 ? 64 : 1];
        float sums[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const float p0 = ex2(fmaf(__uint_as_float(sv[2 * i]), c, shift));
          const float p1 = ex2(fmaf(__uint_as_float(sv[2 * i + 1]), c, shift));
          sums[(2 * i) % 4] += p0;
          sums[(2 * i + 1) % 4] += p1;
          ph[i] = half2_bits(p0, p1);
          if constexpr (TERMS == 2) {
            const float2 back = bits_half2(ph[i]);
            pl[i] = half2_bits(p0 - back.x, p1 - back.y);
          }
        }
        l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          tc::st32(ts + i * 32,
                   *reinterpret_cast<uint32_t(*)[32]>(ph + 32 * i));
          if constexpr (TERMS == 2)
            tc::st32(ts + 64 + i * 32,
                     *reinterpret_cast<uint32_t(*)[32]>(pl + 32 * i));
        }
        // O follows the reference (P_{j-1} V_{j-1} was issued before S_j,
        // which has completed)
        if (j > 0 && __any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int i = 0; i < DIM / 32; ++i) {
            uint32_t ov[32];
            tc::ld32(to + i * 32, ov);
            tc::wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k)
              ov[k] = __float_as_uint(__uint_as_float(ov[k]) * alpha);
            tc::st32(to + i * 32, ov);
          }
        }
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&s.p_full[x]);
      }
      // ---- epilogue
      if (ok)
        ok = wait_all(&s.o_full[x], segments & 1);
      if (!ok)
        break;
      tc::fence_after();
      // (every tile's clearing precedes its P V, which precedes o_full)
      const bool odd = *reinterpret_cast<volatile int*>(&s.odd_values) != 0;
      const bool whole = g.count == g.n_units;
      const int slot = 2 * blockIdx.x + (at > begin ? 1 : 0);
      float* po = a.chunk_part + size_t(slot) * 256 * DIM + (x * 128 + t) * 4;
      float factor = 1;
      if (whole) {
        factor = l > 0 ? 1.0F / l : l == 0 ? 0.0F : l;
        if (a.gate && live)
          factor /= 1 + expf(-to_float(static_cast<const T*>(
                            a.gate)[row * a.ldg + head]));
        if (a.lse && live)
          a.lse[row * a.heads + head] = (m + log2f(l)) * kLn2;
      } else {
        float2* pm = reinterpret_cast<float2*>(
            a.chunk_part + size_t(2 * kChunkCtas) * 256 * DIM);
        pm[slot * 256 + x * 128 + t] = make_float2(m, l);
      }
      T* out = static_cast<T*>(a.out) + row * a.ldo + size_t(head) * DIM;
#pragma unroll
      for (int i = 0; i < DIM / 32; ++i) {
        uint32_t ov[32];
        tc::ld32(to + i * 32, ov);
        tc::wait_ld();
        if (odd && live)
          // values that were cleared although this row sees them
          for (int key = max(oldest, (g.lo_unit + g.u0) * kChunkKeys);
               key <= min(own, (g.lo_unit + g.u0 + g.count) * kChunkKeys - 1);
               ++key) {
            const int k0 = key / kChunkKeys * kChunkKeys;
            if (!(k0 + kChunkKeys - 1 > all_hi || k0 < all_lo))
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
            *reinterpret_cast<uint4*>(po + size_t(i * 8 + k) * 1024) =
                make_uint4(ov[4 * k], ov[4 * k + 1], ov[4 * k + 2],
                           ov[4 * k + 3]);
        } else if (live) {
          alignas(16) T y[32];
#pragma unroll
          for (int k = 0; k < 32; ++k)
            y[k] = from_float<T>(__uint_as_float(ov[k]) * factor);
#pragma unroll
          for (int k = 0; k < 32 * int(sizeof(T)) / 16; ++k)
            reinterpret_cast<uint4*>(out + i * 32)[k] =
                reinterpret_cast<const uint4*>(y)[k];
        }
      }
      if (!whole && g.u0 == 0)
        record = paged_record(at, share, slot, g.n_units, g.q, g.pair, g.h);
      tiles += g.count;
      ++segments;
    }
    if (tid == 0)
      reinterpret_cast<PagedRecord*>(
          a.chunk_part +
          size_t(2 * kChunkCtas) * 256 * (DIM + 2))[blockIdx.x] = record;
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
  if (a.behind_decode)
    grid_dependency_wait();  // this grid ends after the decode kernel's
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
