// Causal GQA attention of a ragged batch over paged keys and values.
// One warp per (row, head), FP32 online softmax over the row's keys.
#include "kernels.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "tensor_map.hpp"

namespace lfm3 {
namespace {

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
  int64_t before;
  const auto none = [](const PagedSequence&) { return int64_t(0); };
  if (!paged_find_row(a.t, none, r, index, s, before) ||
      paged_single(s.n, a.heads / a.t.kv_heads))
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

// Merges the slots of rows that several blocks worked on, writes the rows that
// see no key, leaves the rest. Block = one tensor row, a warp per head at a
// time.
constexpr int kCombineThreads = 128;
template <typename T, int DIM>
__global__ void __launch_bounds__(kCombineThreads)
    paged_combine_kernel(const __grid_constant__ PagedAttentionArgs a) {
  constexpr int kPer = DIM / 32;  // dimensions of a lane
  const int r = blockIdx.x, lane = threadIdx.x % 32;
  const int kvh = a.t.kv_heads, group = a.heads / kvh;
  PagedSequence q{};
  int s;
  int64_t before;
  const auto units = [&](const PagedSequence& x) {
    return int64_t(decode_units(x, group, a.window));
  };
  const bool mine = paged_find_row(a.t, units, r, s, q, before) &&
                    paged_single(q.n, group);
  bool broken;
  const int64_t total = paged_total(a.t, units, broken) * kvh;
  const int64_t share = paged_share(total, kDecodeCtas, kDecodeMinUnits);
  const int n = decode_units(q, group, a.window);
  grid_dependency_wait();  // in every block: this grid ends after the last one
  if (!mine)
    return;
  for (int head = threadIdx.x / 32; head < a.heads;
       head += kCombineThreads / 32) {
    const int h = head / group, j = head % group;
    const int64_t first = before * kvh + int64_t(h) * n;
    const int64_t c0 = first / share, c1 = (first + n - 1) / share;
    if (n > 0 && c0 == c1)
      continue;  // one block had all its keys
    // block c's slot: its first segment unless this one begins inside c
    const auto slot = [&](int64_t c) {
      return 2 * c + (first > c * share ? 1 : 0);
    };
    const float* pm = a.decode_part + size_t(2 * kDecodeCtas) * group * DIM;
    float top = -INFINITY;
    for (int64_t c = c0 + lane; n > 0 && c <= c1; c += 32)
      top = fmaxf(top, pm[(slot(c) * group + j) * 2]);
    top = warp_max(top);
    float l = 0, o[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      o[i] = 0;
#pragma unroll 4
    for (int64_t c = c0; n > 0 && c <= c1; ++c) {
      const int64_t at = slot(c) * group + j;
      const float2 ml = *reinterpret_cast<const float2*>(pm + at * 2);
      const float f = ml.x == -INFINITY ? 0.0F : ex2(ml.x - top);
      l = fmaf(ml.y, f, l);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        o[i] = fmaf(a.decode_part[at * DIM + lane + 32 * i], f, o[i]);
    }
    float scale = n > 0 ? 1.0F / l : 0.0F;
    if (a.gate)
      scale /= 1 + expf(-to_float(
                   static_cast<const T*>(a.gate)[size_t(r) * a.ldg + head]));
    T* out = static_cast<T*>(a.out) + size_t(r) * a.ldo + size_t(head) * DIM;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      out[lane + 32 * i] = from_float<T>(n > 0 ? o[i] * scale : 0.0F);
    if (a.lse && lane == 0)
      a.lse[size_t(r) * a.heads + head] =
          n > 0 ? (top + log2f(l)) * kLn2 : -INFINITY;
  }
}

template <typename T>
cudaError_t launch(PagedAttentionArgs a, uint32_t type, int dim,
                   cudaStream_t stream) {
  const int group = a.heads / a.t.kv_heads;
  const int pool = a.t.pages * a.t.page_rows;
  cudaError_t e;
  if ((e = encode_pool_map(&a.kmap16, a.t.k, pool, a.t.kv_heads, dim, 16,
                           dim / 64)) ||
      (e = encode_pool_map(&a.vmap16, a.t.v, pool, a.t.kv_heads, dim, 16,
                           dim / 64)))
    return e;
  a.decode_part = static_cast<float*>(a.workspace);
  if (group <= kDecodeMaxGroup)
    if ((e = launch_paged_decode(a, type, dim, stream)))
      return e;
  if (!paged_single(a.t.max_rows, group)) {
    const int64_t items = int64_t(a.t.rows) * a.heads;
    if ((e = launch_kernel(dim == 64 ? paged_attention_kernel<T, 64>
                                     : paged_attention_kernel<T, 128>,
                           dim3(unsigned((items + 7) / 8)), dim3(256), 0,
                           stream, false, a)))
      return e;
  }
  return launch_kernel(dim == 64 ? paged_combine_kernel<T, 64>
                                 : paged_combine_kernel<T, 128>,
                       dim3(a.t.rows), dim3(kCombineThreads), 0, stream, true,
                       a);
}

}  // namespace

size_t paged_attention_workspace(const PagedTables& t, int dim, int heads) {
  return paged_decode_floats(dim, heads / t.kv_heads) * 4 + 256;
}

cudaError_t launch_paged_attention(const PagedAttentionArgs& a, uint32_t type,
                                   int dim, cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, type, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, type, dim, stream)
                            : launch<__nv_bfloat16>(a, type, dim, stream);
}

}  // namespace lfm3
