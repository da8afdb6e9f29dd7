// Attention weight per cached key, accumulated. One warp per cached row: its
// key in registers against every query row of the sequence that sees it.
#include "kernels.cuh"
#include "paged.cuh"

namespace lfm3 {
namespace {

template <typename T, int DIM>
__global__ void __launch_bounds__(256)
    paged_key_weights_kernel(const __grid_constant__ PagedKeyWeightsArgs a) {
  constexpr int kPer = DIM / 32;
  const int lane = threadIdx.x % 32;
  const int s = blockIdx.y;
  const PagedSequence q = paged_sequence(a.t, s);
  if (q.broken) {
    report_error(kErrPagedTable);
    return;
  }
  if (q.n == 0)
    return;
  const int group = a.heads / a.t.kv_heads;
  for (int t = blockIdx.x * 8 + threadIdx.x / 32; t < q.length;
       t += gridDim.x * 8) {
    const int pool = paged_row(a.t, a.t.table, s, t);
    if (pool < 0) {
      report_error(kErrPagedTable);
      continue;
    }
    float sum = 0;
    const int base = q.length - q.n;  // number of the first new row
    const int lo = max(0, t - base);
    const int hi = a.window ? min(int64_t(q.n), int64_t(t) - base + a.window)
                            : int64_t(q.n);
    for (int kvh = 0; kvh < a.t.kv_heads; ++kvh) {
      float k[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        k[i] = __half2float(
            a.t.k[(size_t(pool) * a.t.kv_heads + kvh) * DIM + lane * kPer + i]) *
            rsqrtf(float(DIM));
      for (int i = lo; i < hi; ++i)
        for (int g = 0; g < group; ++g) {
          const size_t r = size_t(q.row0 + i);
          const int h = kvh * group + g;
          float x = 0;
#pragma unroll
          for (int d = 0; d < kPer; ++d)
            x += k[d] * to_float(static_cast<const T*>(
                     a.q)[r * a.ldq + size_t(h) * DIM + lane * kPer + d]);
          x = warp_sum(x);
          const float lse = a.lse[r * a.heads + h];
          if (lse != -INFINITY)
            sum += expf(x - lse);
        }
    }
    if (lane == 0)
      a.weights[pool] = t >= base ? sum : a.weights[pool] + sum;
  }
}

template <typename T>
cudaError_t launch(const PagedKeyWeightsArgs& a, int dim, cudaStream_t stream) {
  return launch_kernel(dim == 64 ? paged_key_weights_kernel<T, 64>
                                 : paged_key_weights_kernel<T, 128>,
                       dim3(256, a.t.sequences), dim3(256), 0, stream, false,
                       a);
}

}  // namespace

size_t paged_key_weights_workspace(const PagedTables&, int, int) { return 256; }

cudaError_t launch_paged_key_weights(const PagedKeyWeightsArgs& a,
                                     uint32_t type, int dim,
                                     cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, dim, stream)
                            : launch<__nv_bfloat16>(a, dim, stream);
}

}  // namespace lfm3
