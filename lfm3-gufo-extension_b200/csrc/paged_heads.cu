// Per-head RMSNorm and rotation of a ragged batch's queries and keys, keys and
// values stored in their pages as F16 (lfm3_cuda_paged_heads).
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_i, y_{i + D/2}) turned by position * f_i / c_i,  i < D / 2
//
// An output is then inv (x_i A_i + x_j B_i) with j the partner's place and A_i
// = w_i cos, B_i = -+ w_j sin constants of the row: the partner's raw value is
// all that crosses lanes.
// Every input element is read once and every output written once.
// A thread moves 16 bytes (4 or 8 elements), so a head is 8 to 32 lanes and a
// warp takes 1 to 4 heads at a time; the sum of squares and the partner half
// of each pair come by shuffles inside the head's lanes. Warps are
// independent and stay for several rows: each works on a row, or, when the
// batch has too few rows to fill the GPU, on a part of its heads (a decode
// round: one step of heads a warp). A row's first heads are on their way while
// the warp finds its sequence, page and position and works out its sines and
// cosines, once for all its heads: angle reduced to half turns in FP64 (at
// position 10^5 an FP32 product is off by 2^-8 of a radian), sine and cosine
// of the remainder in FP32.
// Measured: 12868 bf16 rows of 32 + 2 x 8 heads of 64 43.5 us (3.6 TB/s; the
// bytes alone are 24 us). Issue slots are 63 % busy, the ALU 54 %, DRAM 31 %:
// warps wait for fixed latencies and global loads about as long as they work,
// and the partner half of a head is shuffled raw and unpacked a second time. 8
// rows 3.8 us.
#include <algorithm>

#include "kernels.cuh"
#include "paged.cuh"

namespace lfm3 {
namespace {

constexpr int kHeadsThreads = 256;
constexpr int kHeadsWarps = kHeadsThreads / 32;
constexpr int kBlocksPerSm = 3;
constexpr int kWarpsWanted = 148 * kBlocksPerSm * kHeadsWarps;
constexpr int kAhead = 4;               // steps of heads loaded at a time

template <typename T, int DIM>
__global__ void __launch_bounds__(kHeadsThreads, kBlocksPerSm)
    paged_heads_kernel(const __grid_constant__ PagedHeadsArgs a, int parts) {
  constexpr int kVec = 16 / sizeof(T);  // elements of a thread
  constexpr int kLanes = DIM / kVec;    // lanes of a head
  constexpr int kHeadsPerStep = 32 / kLanes;
  constexpr int kHalf = DIM / 2;
  __shared__ float2 turn[kHeadsWarps][kHalf];  // (cos, sin) of each pair
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int sub = lane / kLanes, part = lane % kLanes;
  const int d0 = part * kVec;  // this thread's first element of the head
  const int kvh = a.t.kv_heads;
  // steps of heads: queries, then keys, then values
  const int q_steps = (a.heads + kHeadsPerStep - 1) / kHeadsPerStep;
  const int kv_steps = (kvh + kHeadsPerStep - 1) / kHeadsPerStep;
  const int steps = q_steps + 2 * kv_steps;
  grid_dependency_wait();
  allow_dependents();
  const int64_t units = int64_t(a.t.rows) * parts;
  const int64_t stride = int64_t(gridDim.x) * kHeadsWarps;
  int64_t unit = int64_t(blockIdx.x) * kHeadsWarps + warp;
  if (unit >= units)
    return;
  int r, first;  // the warp's row, and which of its parts
  uint4 raw[kAhead];
  // step's kind (0 queries, 1 keys, 2 values) and this lane's head of it
  const auto kind_of = [&](int step) {
    return step < q_steps ? 0 : step < q_steps + kv_steps ? 1 : 2;
  };
  const auto head_of = [&](int step, int kind) {
    return (step - (kind ? q_steps : 0) - (kind == 2 ? kv_steps : 0)) *
               kHeadsPerStep + sub;
  };
  const T *q_row, *k_row, *v_row;  // of row r, from element d0 on
  const auto load = [&](int step0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int step = step0 + i * parts, kind = kind_of(step);
      const int h = head_of(step, kind);
      const T* base = kind == 0 ? q_row : kind == 1 ? k_row : v_row;
      if (step < steps && h < (kind ? kvh : a.heads))
        raw[i] = *reinterpret_cast<const uint4*>(base + h * DIM);
    }
  };
  const auto begin = [&]() {
    // (with several parts a row, rows are few)
    r = parts == 1 ? int(unit) : int(uint32_t(unit) / uint32_t(parts));
    first = int(unit - int64_t(r) * parts);
    q_row = static_cast<const T*>(a.q) + size_t(r) * a.ldq + d0;
    k_row = static_cast<const T*>(a.k) + size_t(r) * a.ldk + d0;
    v_row = static_cast<const T*>(a.v) + size_t(r) * a.ldv + d0;
    load(first);
  };
  begin();
  // ---- constants of the warp: the first 32 sequences, a lane each, the
  // pairs' half turns per position, this lane's norm weights
  PagedSequence mine{0, 0, 0, true};
  if (lane < a.t.sequences)
    mine = paged_sequence(a.t, lane);
  if (unit == 0)
    for (int s = lane; s < a.t.sequences; s += 32)
      if (paged_sequence(a.t, s).broken)
        report_error(kErrPagedTable);
  double turns[kHalf / 32];
#pragma unroll
  for (int i = 0; i < kHalf / 32; ++i) {
    turns[i] = double(a.freq[lane + 32 * i]) * 0.31830988618379067154;  // 1/pi
    if (a.factors)
      turns[i] /= double(a.factors[lane + 32 * i]);
  }
  // norm weights of this lane's elements and of their partners
  const int other = (d0 + kHalf) % DIM;
  const float sign = d0 < kHalf ? -1.0F : 1.0F;

  for (;;) {
    // ---- the sequence that holds tensor row r
    int s = -1, number = 0;
    for (int s0 = 0; s0 < a.t.sequences && s < 0; s0 += 32) {
      PagedSequence q = mine;
      if (s0 > 0) {
        q = PagedSequence{0, 0, 0, true};
        if (s0 + lane < a.t.sequences)
          q = paged_sequence(a.t, s0 + lane);
      }
      const unsigned any = __ballot_sync(
          0xffffffffu, !q.broken && r >= q.row0 && r < q.row0 + q.n);
      if (any) {
        const int l = __ffs(any) - 1;
        s = s0 + l;
        number = __shfl_sync(0xffffffffu, q.length - q.n - q.row0, l) + r;
      }
    }
    if (s >= 0) {  // else not a row of the batch
      int pool = -1;
      if (number >= 0) {
        pool = paged_row(a.t, a.t.table, s, number);
        if (pool < 0 && lane == 0)
          report_error(kErrPagedTable);
      }
      const int position = a.positions ? a.positions[r] : number;
#pragma unroll
      for (int i = 0; i < kHalf / 32; ++i) {
        const double t = double(position) * turns[i];
        float sn, cs;
        sincospif(float(t - 2.0 * rint(t * 0.5)), &sn, &cs);
        turn[warp][lane + 32 * i] = make_float2(cs, sn);
      }
      __syncwarp();
      F32x2 fa[kVec / 2], fb[kVec / 2];  // A and B of this lane's elements
      int factors_of = -1;
      T* const q_out = static_cast<T*>(a.q_out) + size_t(r) * a.ldo + d0;
      const size_t page_row = size_t(max(pool, 0)) * kvh * DIM + d0;
      for (int step0 = first; step0 < steps; step0 += kAhead * parts) {
        if (step0 != first)
          load(step0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int step = step0 + i * parts, kind = kind_of(step);
          const int h = head_of(step, kind);
          const bool live = h < (kind ? kvh : a.heads);
          const float* w = kind ? a.k_norm : a.q_norm;
          if (step >= steps)
            continue;
          float x[kVec];
          unpack16(raw[i], x, T{});
          if (kind < 2) {
            if (kind != factors_of) {
              factors_of = kind;
#pragma unroll
              for (int k = 0; k < kVec; k += 2) {
                const float2 t0 = turn[warp][(d0 + k) % kHalf];
                const float2 t1 = turn[warp][(d0 + k + 1) % kHalf];
                const float a0 = w ? w[d0 + k] : 1.0F;
                const float a1 = w ? w[d0 + k + 1] : 1.0F;
                const float b0 = w ? w[other + k] : 1.0F;
                const float b1 = w ? w[other + k + 1] : 1.0F;
                fa[k / 2] = pair(a0 * t0.x, a1 * t1.x);
                fb[k / 2] = pair(sign * b0 * t0.y, sign * b1 * t1.y);
              }
            }
            uint4 across;
            across.x = __shfl_xor_sync(0xffffffffu, raw[i].x, kLanes / 2);
            across.y = __shfl_xor_sync(0xffffffffu, raw[i].y, kLanes / 2);
            across.z = __shfl_xor_sync(0xffffffffu, raw[i].z, kLanes / 2);
            across.w = __shfl_xor_sync(0xffffffffu, raw[i].w, kLanes / 2);
            float o[kVec];
            unpack16(across, o, T{});
            F32x2 sum2 = pair(0, 0), y[kVec / 2];
#pragma unroll
            for (int k = 0; k < kVec / 2; ++k) {
              const F32x2 v = pair(x[2 * k], x[2 * k + 1]);
              sum2 = fma_pair(v, v, sum2);
              y[k] = fma_pair(v, fa[k],
                              mul_pair(pair(o[2 * k], o[2 * k + 1]), fb[k]));
            }
            const float2 sums = both(sum2);
            float squares = sums.x + sums.y;
#pragma unroll
            for (int n = kLanes / 2; n; n >>= 1)
              squares += __shfl_xor_sync(0xffffffffu, squares, n);
            const float inv =
                w ? rsqrtf(squares * (1.0F / DIM) + a.eps) : 1.0F;
            const F32x2 inv2 = pair(inv, inv);
#pragma unroll
            for (int k = 0; k < kVec / 2; ++k) {
              const float2 v = both(mul_pair(y[k], inv2));
              x[2 * k] = v.x;
              x[2 * k + 1] = v.y;
            }
          }
          if (kind == 0) {
            if (live)
              *reinterpret_cast<uint4*>(q_out + h * DIM) = pack16(x, T{});
          } else if (live && pool >= 0) {
            __half* dst = (kind == 1 ? a.t.k : a.t.v) + page_row + h * DIM;
            if constexpr (kVec == 8)
              *reinterpret_cast<uint4*>(dst) = pack16(x, __half{});
            else
              *reinterpret_cast<uint2*>(dst) =
                  make_uint2(pack2(x[0], x[1], __half{}),
                             pack2(x[2], x[3], __half{}));
          }
        }
      }
      __syncwarp();  // turn is written again
    }
    unit += stride;
    if (unit >= units)
      return;
    begin();
  }
}

template <typename T, int DIM>
cudaError_t launch(const PagedHeadsArgs& a, cudaStream_t stream) {
  const int per = 32 / (DIM * int(sizeof(T)) / 16);
  const int steps = (a.heads + per - 1) / per +
                    2 * ((a.t.kv_heads + per - 1) / per);
  int parts = (kWarpsWanted + a.t.rows - 1) / a.t.rows;
  parts = parts < steps ? parts : steps;
  const int64_t warps = int64_t(a.t.rows) * parts;
  const int64_t blocks = std::min<int64_t>(
      (warps + kHeadsWarps - 1) / kHeadsWarps, 148 * kBlocksPerSm);
  return launch_kernel(paged_heads_kernel<T, DIM>, dim3(unsigned(blocks)),
                       dim3(kHeadsThreads), 0, stream, true, a, parts);
}
template <typename T>
cudaError_t launch(const PagedHeadsArgs& a, int dim, cudaStream_t stream) {
  return dim == 64 ? launch<T, 64>(a, stream) : launch<T, 128>(a, stream);
}

}  // namespace

cudaError_t launch_paged_heads(const PagedHeadsArgs& a, uint32_t type, int dim,
                               cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, dim, stream)
                            : launch<__nv_bfloat16>(a, dim, stream);
}

}  // namespace lfm3
