// Per-head RMSNorm and rotation of a ragged batch's queries and keys, keys and
// values stored in their pages as F16 (lfm3_cuda_paged_heads).
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_i, y_{i + D/2}) turned by position * f_i / c_i,  i < D / 2
//
// HBM bound: every input element is read once and every output written once.
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
  const int kvh = a.t.kv_heads, all = a.heads + 2 * kvh;
  const int steps = (all + kHeadsPerStep - 1) / kHeadsPerStep;
  grid_dependency_wait();
  allow_dependents();
  const int64_t units = int64_t(a.t.rows) * parts;
  const int64_t stride = int64_t(gridDim.x) * kHeadsWarps;
  int64_t unit = int64_t(blockIdx.x) * kHeadsWarps + warp;
  if (unit >= units)
    return;
  int r, first;  // the warp's row, and which of its parts
  uint4 raw[kAhead];
  const auto load = [&](int step0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = (step0 + i * parts) * kHeadsPerStep + sub;
      // queries, then keys, then values
      const T* src =
          h < a.heads ? static_cast<const T*>(a.q) + size_t(r) * a.ldq +
                            size_t(h) * DIM
          : h < a.heads + kvh
              ? static_cast<const T*>(a.k) + size_t(r) * a.ldk +
                    size_t(h - a.heads) * DIM
              : static_cast<const T*>(a.v) + size_t(r) * a.ldv +
                    size_t(h - a.heads - kvh) * DIM;
      if (h < all)
        raw[i] = *reinterpret_cast<const uint4*>(src + d0);
    }
  };
  const auto begin = [&]() {
    r = int(unit / parts);
    first = int(unit - int64_t(r) * parts);
    load(first);
  };
  begin();
  // ---- constants of the warp: the first 32 sequences, a lane each, the
  // pairs' half turns per position, this lane's norm weights
  PagedSequence mine{0, 0, 0, true};
  if (lane < a.t.sequences) {
    mine = paged_sequence(a.t, lane);
    if (mine.broken && unit == 0)
      report_error(kErrPagedTable);
  }
  double turns[kHalf / 32];
#pragma unroll
  for (int i = 0; i < kHalf / 32; ++i) {
    turns[i] = double(a.freq[lane + 32 * i]) * 0.31830988618379067154;  // 1/pi
    if (a.factors)
      turns[i] /= double(a.factors[lane + 32 * i]);
  }
  float wq[kVec];
#pragma unroll
  for (int k = 0; k < kVec; ++k)
    wq[k] = a.q_norm ? a.q_norm[d0 + k] : 1.0F;

  for (;;) {
    // ---- the sequence that holds tensor row r
    int s = -1, number = 0;
    for (int s0 = 0; s0 < a.t.sequences && s < 0; s0 += 32) {
      PagedSequence q = mine;
      if (s0 > 0) {
        q = PagedSequence{0, 0, 0, true};
        if (s0 + lane < a.t.sequences) {
          q = paged_sequence(a.t, s0 + lane);
          if (q.broken && unit == 0)
            report_error(kErrPagedTable);
        }
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
      float cs[kVec], sn[kVec];  // of this lane's pairs; + for the second half
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const float2 t = turn[warp][(d0 + k) % kHalf];
        cs[k] = t.x;
        sn[k] = d0 < kHalf ? -t.y : t.y;
      }
      __syncwarp();
      for (int step0 = first; step0 < steps; step0 += kAhead * parts) {
        if (step0 != first)
          load(step0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (step0 + i * parts >= steps)
            break;
          const int h = (step0 + i * parts) * kHeadsPerStep + sub;
          const bool live = h < all, query = h < a.heads;
          const bool value = h >= a.heads + kvh;
          const T* e = reinterpret_cast<const T*>(&raw[i]);
          float x[kVec], y[kVec];
          float squares = 0;
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            x[k] = live ? to_float(e[k]) : 0.0F;
            squares += x[k] * x[k];
          }
#pragma unroll
          for (int o = kLanes / 2; o; o >>= 1)
            squares += __shfl_xor_sync(0xffffffffu, squares, o);
          const bool norm = query ? a.q_norm != nullptr : a.k_norm != nullptr;
          const float inv =
              norm ? 1.0F / sqrtf(squares * (1.0F / DIM) + a.eps) : 1.0F;
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            const float w = query  ? wq[k]
                            : norm ? a.k_norm[d0 + k]
                                   : 1.0F;
            const float n = (x[k] * inv) * w;
            const float other = __shfl_xor_sync(0xffffffffu, n, kLanes / 2);
            // first half: a cos - b sin; second half: b cos + a sin
            y[k] = n * cs[k] + other * sn[k];
          }
          if (!live)
            continue;
          if (query) {
            alignas(16) T out[kVec];
#pragma unroll
            for (int k = 0; k < kVec; ++k)
              out[k] = from_float<T>(y[k]);
            *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) +
                                      size_t(r) * a.ldo + size_t(h) * DIM +
                                      d0) =
                *reinterpret_cast<const uint4*>(out);
          } else if (pool >= 0) {
            alignas(16) __half out[kVec];
#pragma unroll
            for (int k = 0; k < kVec; ++k)
              out[k] = __float2half_rn(value ? x[k] : y[k]);
            __half* dst = (value ? a.t.v : a.t.k) +
                          (size_t(pool) * kvh +
                           (value ? h - a.heads - kvh : h - a.heads)) *
                              DIM +
                          d0;
            if constexpr (kVec == 8)
              *reinterpret_cast<uint4*>(dst) =
                  *reinterpret_cast<const uint4*>(out);
            else
              *reinterpret_cast<uint2*>(dst) =
                  *reinterpret_cast<const uint2*>(out);
          }
        }
      }
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
  const int steps = (a.heads + 2 * a.t.kv_heads + per - 1) / per;
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
