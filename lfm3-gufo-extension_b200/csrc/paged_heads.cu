// Per-head RMSNorm and rotation of a ragged batch's queries and keys, keys and
// values stored in their pages as F16 (lfm3_cuda_paged_heads).
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_i, y_{i + D/2}) turned by position * f_i / c_i,  i < D / 2
//
// HBM bound: every input element is read once and every output written once.
// A thread moves 16 bytes (4 or 8 elements), so a head is 8 to 32 lanes and a
// warp takes 1 to 4 heads at a time; the sum of squares and the partner half
// of each pair come by shuffles inside the head's lanes. A block takes whole
// rows: its first D / 2 threads turn the row's position into sines and
// cosines once for all heads. The angle is reduced to half turns in FP64 (at
// position 10^5 an FP32 product is off by 2^-8 of a radian), the sine and
// cosine of the remainder are FP32.
#include "kernels.cuh"
#include "paged.cuh"

namespace lfm3 {
namespace {

constexpr int kHeadsThreads = 256;
constexpr int kHeadsBlocks = 148 * 8;  // resident blocks of a B200

template <typename T, int DIM>
__global__ void __launch_bounds__(kHeadsThreads)
    paged_heads_kernel(const __grid_constant__ PagedHeadsArgs a) {
  constexpr int kVec = 16 / sizeof(T);        // elements of a thread
  constexpr int kLanes = DIM / kVec;          // lanes of a head
  constexpr int kHeadsPerWarp = 32 / kLanes;
  constexpr int kHalf = DIM / 2;
  __shared__ float cs[kHalf], sn[kHalf];
  __shared__ int where[3];  // sequence (-1: none), row number, tensor row
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int sub = lane / kLanes, part = lane % kLanes;
  const int d0 = part * kVec;  // this thread's first element of the head
  const int kvh = a.t.kv_heads, all = a.heads + 2 * kvh;
  double turns = 0;  // half turns per position of pair tid
  if (tid < kHalf) {
    double f = double(a.freq[tid]);
    if (a.factors)
      f /= double(a.factors[tid]);
    turns = f * 0.31830988618379067154;  // 1 / pi
  }
  for (int r = blockIdx.x; r < a.t.rows; r += gridDim.x) {
    if (warp == 0) {
      // the sequence that holds tensor row r
      int found = -1, number = 0;
      for (int s0 = 0; s0 < a.t.sequences && found < 0; s0 += 32) {
        const int s = s0 + lane;
        bool hit = false;
        int row = 0;
        if (s < a.t.sequences) {
          const PagedSequence q = paged_sequence(a.t, s);
          hit = !q.broken && r >= q.row0 && r < q.row0 + q.n;
          row = q.length - q.n + (r - q.row0);
          if (q.broken && r == blockIdx.x)
            report_error(kErrPagedTable);
        }
        const unsigned any = __ballot_sync(0xffffffffu, hit);
        if (any) {
          found = s0 + __ffs(any) - 1;
          number = __shfl_sync(0xffffffffu, row, __ffs(any) - 1);
        }
      }
      if (lane == 0) {
        where[0] = found;
        where[1] = number;
        int pool = -1;
        if (found >= 0 && number >= 0) {
          pool = paged_row(a.t, a.t.table, found, number);
          if (pool < 0)
            report_error(kErrPagedTable);
        }
        where[2] = pool;
      }
    }
    __syncthreads();
    const int s = where[0], pool = where[2];
    if (s >= 0 && tid < kHalf) {
      const int position = a.positions ? a.positions[r] : where[1];
      const double t = double(position) * turns;
      sincospif(float(t - 2.0 * rint(t * 0.5)), &sn[tid], &cs[tid]);
    }
    __syncthreads();
    if (s >= 0) {
      for (int h0 = warp * kHeadsPerWarp; h0 < all;
           h0 += kHeadsThreads / 32 * kHeadsPerWarp) {
        const int h = h0 + sub;  // queries, then keys, then values
        const bool live = h < all, query = h < a.heads;
        const bool value = h >= a.heads + kvh;
        const int kh = value ? h - a.heads - kvh : h - a.heads;
        float x[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          x[i] = 0;
        if (live) {
          const T* src =
              query   ? static_cast<const T*>(a.q) + size_t(r) * a.ldq + size_t(h) * DIM
              : value ? static_cast<const T*>(a.v) + size_t(r) * a.ldv + size_t(kh) * DIM
                      : static_cast<const T*>(a.k) + size_t(r) * a.ldk + size_t(kh) * DIM;
          alignas(16) T raw[kVec];
          *reinterpret_cast<uint4*>(raw) =
              *reinterpret_cast<const uint4*>(src + d0);
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            x[i] = to_float(raw[i]);
        }
        float y[kVec];
        const float* w = query ? a.q_norm : a.k_norm;
        float squares = 0;
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          squares += x[i] * x[i];
#pragma unroll
        for (int o = kLanes / 2; o; o >>= 1)
          squares += __shfl_xor_sync(0xffffffffu, squares, o);
        const float inv = 1.0F / sqrtf(squares * (1.0F / DIM) + a.eps);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float n = w ? (x[i] * inv) * w[d0 + i] : x[i];
          const float other = __shfl_xor_sync(0xffffffffu, n, kLanes / 2);
          const int p = (d0 + i) % kHalf;
          // first half: a cos - b sin; second half: b cos + a sin
          y[i] = d0 < kHalf ? n * cs[p] - other * sn[p]
                            : n * cs[p] + other * sn[p];
        }
        if (!live)
          continue;
        if (query) {
          alignas(16) T raw[kVec];
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            raw[i] = from_float<T>(y[i]);
          *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) +
                                    size_t(r) * a.ldo + size_t(h) * DIM + d0) =
              *reinterpret_cast<const uint4*>(raw);
        } else if (pool >= 0) {
          alignas(16) __half raw[kVec];
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            raw[i] = __float2half_rn(value ? x[i] : y[i]);
          __half* dst = (value ? a.t.v : a.t.k) +
                        (size_t(pool) * kvh + kh) * DIM + d0;
          if constexpr (kVec == 8)
            *reinterpret_cast<uint4*>(dst) =
                *reinterpret_cast<const uint4*>(raw);
          else
            *reinterpret_cast<uint2*>(dst) =
                *reinterpret_cast<const uint2*>(raw);
        }
      }
    }
    __syncthreads();  // where, cs and sn are written again
  }
}

template <typename T>
cudaError_t launch(const PagedHeadsArgs& a, int dim, cudaStream_t stream) {
  const dim3 grid(a.t.rows < kHeadsBlocks ? a.t.rows : kHeadsBlocks);
  return launch_kernel(dim == 64 ? paged_heads_kernel<T, 64>
                                 : paged_heads_kernel<T, 128>,
                       grid, dim3(kHeadsThreads), 0, stream, false, a);
}

}  // namespace

cudaError_t launch_paged_heads(const PagedHeadsArgs& a, uint32_t type, int dim,
                               cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, dim, stream)
                            : launch<__nv_bfloat16>(a, dim, stream);
}

}  // namespace lfm3
