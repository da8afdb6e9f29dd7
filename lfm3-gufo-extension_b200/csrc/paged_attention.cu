// Causal GQA attention of a ragged batch over paged keys and values.
// One warp per (row, head), FP32 online softmax over the row's keys.
#include "kernels.cuh"
#include "paged.cuh"

namespace lfm3 {
namespace {

// The sequence that holds tensor row r (warp-wide), false if none does.
__device__ bool find_row(const PagedTables& t, int r, PagedSequence& out,
                         int& index) {
  const int lane = threadIdx.x % 32;
  for (int s0 = 0; s0 < t.sequences; s0 += 32) {
    PagedSequence q{0, 0, 0, true};
    if (s0 + lane < t.sequences) {
      q = paged_sequence(t, s0 + lane);
      if (q.broken)
        report_error(kErrPagedTable);
    }
    const unsigned any = __ballot_sync(
        0xffffffffu, !q.broken && r >= q.row0 && r < q.row0 + q.n);
    if (any) {
      const int l = __ffs(any) - 1;
      index = s0 + l;
      out.row0 = __shfl_sync(0xffffffffu, q.row0, l);
      out.n = __shfl_sync(0xffffffffu, q.n, l);
      out.length = __shfl_sync(0xffffffffu, q.length, l);
      return true;
    }
  }
  return false;
}

template <typename T, int DIM>
__global__ void __launch_bounds__(256)
    paged_attention_kernel(const __grid_constant__ PagedAttentionArgs a) {
  constexpr int kPer = DIM / 32;
  const int lane = threadIdx.x % 32;
  const int64_t item = int64_t(blockIdx.x) * 8 + threadIdx.x / 32;
  const int r = int(item / a.heads), h = int(item % a.heads);
  if (r >= a.t.rows)
    return;
  PagedSequence s{};
  int index = 0;
  if (!find_row(a.t, r, s, index))
    return;
  const int own = s.length - s.n + (r - s.row0);
  const int first = a.window ? max(0, own - a.window + 1) : 0;
  const int kvh = h / (a.heads / a.t.kv_heads);
  float q[kPer], o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    q[i] = to_float(static_cast<const T*>(a.q)[size_t(r) * a.ldq +
                                               size_t(h) * DIM + lane * kPer + i]) *
           rsqrtf(float(DIM));
    o[i] = 0;
  }
  float m = -INFINITY, l = 0;
  for (int t = first; t <= own; ++t) {
    const int pool = paged_row(a.t, a.t.table, index, t);
    if (pool < 0) {
      report_error(kErrPagedTable);
      continue;
    }
    const size_t at = (size_t(pool) * a.t.kv_heads + kvh) * DIM + lane * kPer;
    float x = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      x += q[i] * __half2float(a.t.k[at + i]);
    x = warp_sum(x);
    const float top = fmaxf(m, x);
    const float alpha = expf(m - top), p = expf(x - top);
    m = top;
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      o[i] = o[i] * alpha + p * __half2float(a.t.v[at + i]);
  }
  const bool empty = own < first;
  float scale = empty ? 0.0F : 1.0F / l;
  if (a.gate)
    scale /= 1 + expf(-to_float(static_cast<const T*>(a.gate)[size_t(r) * a.ldg + h]));
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    static_cast<T*>(a.out)[size_t(r) * a.ldo + size_t(h) * DIM + lane * kPer + i] =
        from_float<T>(empty ? 0.0F : o[i] * scale);
  if (a.lse && lane == 0)
    a.lse[size_t(r) * a.heads + h] = empty ? -INFINITY : m + logf(l);
}

template <typename T>
cudaError_t launch(const PagedAttentionArgs& a, int dim, cudaStream_t stream) {
  const int64_t items = int64_t(a.t.rows) * a.heads;
  return launch_kernel(dim == 64 ? paged_attention_kernel<T, 64>
                                 : paged_attention_kernel<T, 128>,
                       dim3(unsigned((items + 7) / 8)), dim3(256), 0, stream,
                       false, a);
}

}  // namespace

size_t paged_attention_workspace(const PagedTables&, int, int) { return 256; }

cudaError_t launch_paged_attention(const PagedAttentionArgs& a, uint32_t type,
                                   int dim, cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, dim, stream)
                            : launch<__nv_bfloat16>(a, dim, stream);
}

}  // namespace lfm3
