// Causal GQA attention of a ragged batch over paged keys and values: single
// tokens on paged_decode.cu, every other sequence on paged_chunk.cu, and the
// merge of rows whose keys several blocks shared.
#include <algorithm>

#include "kernels.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "tensor_map.hpp"

namespace lfm3 {
namespace {

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
  int64_t before = 0, total = 0, share = 0, first_unit = 0;
  int n = 0;       // key units of the row's tile and KV head
  int trow = 0;    // chunk: the row's place in its pair of row tiles
  bool broken, single = false;
  const auto decode = [&](const PagedSequence& x) {
    return int64_t(decode_units(x, group, a.window));
  };
  const auto chunk = [&](const PagedSequence& x) {
    return chunk_sequence_units(x, group, a.window);
  };
  bool mine = paged_find_row(a.t, decode, r, s, q, before);
  if (mine && paged_single(q.n, group)) {
    single = true;
    n = decode_units(q, group, a.window);
    total = paged_total(a.t, decode, broken) * kvh;
    share = paged_share(total, kDecodeCtas, kDecodeMinUnits);
    first_unit = before * kvh;
  } else if (mine) {
    mine = paged_find_row(a.t, chunk, r, s, q, before);
    const int queries = 2 * chunk_queries(group), i = r - q.row0;
    int lo;
    for (int p = 0; p < i / queries; ++p)
      before += chunk_units(q, group, a.window, p, lo);
    n = chunk_units(q, group, a.window, i / queries, lo);
    trow = i % queries / (queries / 2) * kChunkRows +
           i % (queries / 2) * group;
    total = paged_total(a.t, chunk, broken) * kvh;
    share = paged_share(total, kChunkCtas, kChunkMinUnits);
    first_unit = before * kvh;
  }
  grid_dependency_wait();  // in every block: this grid ends after the last one
  if (!mine)
    return;
  const float* part = single ? a.decode_part : a.chunk_part;
  const float* pm =
      part + (single ? size_t(2 * kDecodeCtas) * group * DIM
                     : size_t(2 * kChunkCtas) * 2 * kChunkRows * DIM);
  for (int head = threadIdx.x / 32; head < a.heads;
       head += kCombineThreads / 32) {
    const int h = head / group, j = head % group;
    const int64_t first = first_unit + int64_t(h) * n;
    const int64_t c0 = first / share, c1 = (first + n - 1) / share;
    if (n > 0 && c0 == c1)
      continue;  // one block had all its keys
    // block c's slot: its first segment unless this one begins inside c
    const auto slot = [&](int64_t c) {
      return 2 * c + (first > c * share ? 1 : 0);
    };
    // its entry of (max, sum), and this lane's four output values
    const auto entry = [&](int64_t c) {
      return single ? slot(c) * group + j
                    : slot(c) * (2 * kChunkRows) + trow + j;
    };
    const auto values = [&](int64_t c) {
      return single ? part + entry(c) * DIM + lane * 4
                    : part + slot(c) * (2 * kChunkRows) * DIM +
                          (lane * (2 * kChunkRows) + trow + j) * 4;
    };
    float top = -INFINITY;
    for (int64_t c = c0 + lane; n > 0 && c <= c1; c += 32)
      top = fmaxf(top, pm[entry(c) * 2]);
    top = warp_max(top);
    float l = 0, o[4] = {0, 0, 0, 0};
#pragma unroll 4
    for (int64_t c = c0; n > 0 && c <= c1; ++c) {
      const float2 ml = *reinterpret_cast<const float2*>(pm + entry(c) * 2);
      float4 v = make_float4(0, 0, 0, 0);
      if (lane < DIM / 4)
        v = *reinterpret_cast<const float4*>(values(c));
      if (ml.x == -INFINITY && ml.y == 0)
        continue;  // no visible key there
      const float f = ml.x == -INFINITY ? 1.0F : ex2(ml.x - top);
      l = fmaf(ml.y, f, l);
      o[0] = fmaf(v.x, f, o[0]);
      o[1] = fmaf(v.y, f, o[1]);
      o[2] = fmaf(v.z, f, o[2]);
      o[3] = fmaf(v.w, f, o[3]);
    }
    const bool empty = l == 0;
    float scale = empty ? 0.0F : 1.0F / l;
    if (a.gate)
      scale /= 1 + expf(-to_float(
                   static_cast<const T*>(a.gate)[size_t(r) * a.ldg + head]));
    T* out = static_cast<T*>(a.out) + size_t(r) * a.ldo + size_t(head) * DIM;
    if (lane < DIM / 4) {
      alignas(16) T y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[i] = from_float<T>(empty ? 0.0F : o[i] * scale);
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<uint4*>(out + lane * 4) =
            *reinterpret_cast<const uint4*>(y);
      else
        *reinterpret_cast<uint2*>(out + lane * 4) =
            *reinterpret_cast<const uint2*>(y);
    }
    if (a.lse && lane == 0)
      a.lse[size_t(r) * a.heads + head] =
          empty ? -INFINITY : (top + log2f(l)) * kLn2;
  }
}

template <typename T>
cudaError_t launch(PagedAttentionArgs a, uint32_t type, int dim,
                   cudaStream_t stream) {
  const int group = a.heads / a.t.kv_heads;
  const int pool = a.t.pages * a.t.page_rows;
  cudaError_t e;
  a.decode_part = static_cast<float*>(a.workspace);
  a.chunk_part = a.decode_part + paged_decode_floats(dim, group);
  if (group <= kDecodeMaxGroup) {
    if ((e = encode_pool_map(&a.kmap16, a.t.k, pool, a.t.kv_heads, dim, 16,
                             dim / 64)) ||
        (e = encode_pool_map(&a.vmap16, a.t.v, pool, a.t.kv_heads, dim, 16,
                             dim / 64)) ||
        (e = launch_paged_decode(a, type, dim, stream)))
      return e;
  }
  if (!paged_single(a.t.max_rows, group)) {
    // the largest box that never crosses a page
    a.box_rows = std::min(a.t.page_rows & -a.t.page_rows, kChunkKeys);
    if ((e = encode_pool_map(&a.kmap, a.t.k, pool, a.t.kv_heads, dim,
                             a.box_rows, 1)) ||
        (e = encode_pool_map(&a.vmap, a.t.v, pool, a.t.kv_heads, dim,
                             a.box_rows, 1)) ||
        (e = launch_paged_chunk(a, type, dim, stream)))
      return e;
  }
  return launch_kernel(dim == 64 ? paged_combine_kernel<T, 64>
                                 : paged_combine_kernel<T, 128>,
                       dim3(a.t.rows), dim3(kCombineThreads), 0, stream, true,
                       a);
}

}  // namespace

size_t paged_attention_workspace(const PagedTables& t, int dim, int heads) {
  const int group = heads / t.kv_heads;
  return (paged_decode_floats(dim, group) +
          (paged_single(t.max_rows, group) ? 0 : paged_chunk_floats(dim))) * 4;
}

cudaError_t launch_paged_attention(const PagedAttentionArgs& a, uint32_t type,
                                   int dim, cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, type, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, type, dim, stream)
                            : launch<__nv_bfloat16>(a, type, dim, stream);
}

}  // namespace lfm3
