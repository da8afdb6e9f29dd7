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

// Two partial rows (maximum, sum) as one; a sum without a maximum is 0, or
// NaN, which has to stay. Returns the factors of their outputs.
__device__ __forceinline__ float2 merge(float2& a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  const float fa = a.x == -INFINITY ? 1.0F : ex2(a.x - m);
  const float fb = b.x == -INFINITY ? 1.0F : ex2(b.x - m);
  a = make_float2(m, a.y * fa + b.y * fb);
  return make_float2(fa, fb);
}

// Merges the stretches that several blocks shared: the decode kernel's records
// (a single token's G heads), a head a warp, then the chunk kernel's, 32 of a
// record's 256 rows a block at a time (only some of its 148 blocks leave one).
// Slots add up in key order.
constexpr int kCombineRows = 32;

template <typename T, int DIM>
__device__ void combine_single(const PagedAttentionArgs& a) {
  constexpr int kAhead = 16;  // slots whose loads are in flight at once
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int group = a.heads / a.t.kv_heads;
  const float2* pm = reinterpret_cast<const float2*>(
      a.decode_part + size_t(2 * kDecodeCtas) * group * DIM);
  const PagedRecord* records = reinterpret_cast<const PagedRecord*>(
      pm + size_t(2 * kDecodeCtas) * group);
  const int warps = blockDim.x / 32;
  // a warp a head, a lane four dimensions
  for (int u = blockIdx.x * warps + warp; u < kDecodeCtas * group;
       u += gridDim.x * warps) {
    const PagedRecord rec = records[u / group];
    const int j = u % group;
    if (rec.parts == 0)
      continue;
    const float* src = a.decode_part + size_t(j) * DIM + lane % (DIM / 4) * 4;
    const int head = rec.h * group + j;
    float gate = INFINITY;
    if (a.gate)
      gate = to_float(static_cast<const T*>(
          a.gate)[size_t(rec.row0) * a.ldg + head]);
    float2 ml = make_float2(-INFINITY, 0);
    float4 o = make_float4(0, 0, 0, 0);
    for (int p0 = 0; p0 < rec.parts; p0 += kAhead) {
      float4 v[kAhead];
      float2 b[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int sl = record_slot(rec, min(p0 + k, rec.parts - 1));
        b[k] = pm[sl * group + j];
        v[k] = *reinterpret_cast<const float4*>(src + size_t(sl) * group * DIM);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (p0 + k >= rec.parts)
          break;
        const float2 f = merge(ml, b[k]);
        o.x = o.x * f.x + v[k].x * f.y;
        o.y = o.y * f.x + v[k].y * f.y;
        o.z = o.z * f.x + v[k].z * f.y;
        o.w = o.w * f.x + v[k].w * f.y;
      }
    }
    // (a sum of 0: no key but scores of -inf, a row like one without keys)
    const float scale = ml.y == 0 ? 0.0F : 1.0F / ml.y / (1 + expf(-gate));
    T* out = static_cast<T*>(a.out) + size_t(rec.row0) * a.ldo +
             size_t(head) * DIM + lane * 4;
    if (lane < DIM / 4) {
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(out) =
            make_float4(o.x * scale, o.y * scale, o.z * scale, o.w * scale);
      else
        *reinterpret_cast<uint2*>(out) =
            make_uint2(pack2(o.x * scale, o.y * scale, T{}),
                       pack2(o.z * scale, o.w * scale, T{}));
    }
    if (a.lse && lane == 0)
      a.lse[size_t(rec.row0) * a.heads + head] = (ml.x + log2f(ml.y)) * kLn2;
  }
}

template <typename T, int DIM>
__device__ void combine_chunks(const PagedAttentionArgs& a) {
  constexpr int kRows = 2 * kChunkRows;  // of a slot
  constexpr int kQuads = DIM / 4, kAhead = 8;
  constexpr int kThreads = 512;
  static_assert(kThreads >= 8 * kCombineRows && kChunkCtas <= kThreads);
  alignas(16) __shared__ float tile[kCombineRows][DIM + 4];
  __shared__ float2 row_scales[kCombineRows];  // maximum, factor
  __shared__ int list[kChunkCtas];             // blocks that left a record
  __shared__ int listed;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int group = a.heads / a.t.kv_heads, QB = chunk_queries(group);
  const float2* pm = reinterpret_cast<const float2*>(
      a.chunk_part + size_t(2 * kChunkCtas) * kRows * DIM);
  const PagedRecord* records = reinterpret_cast<const PagedRecord*>(
      pm + size_t(2 * kChunkCtas) * kRows);
  if (warp == 0) {
    int count = 0;
    for (int b0 = 0; b0 < kChunkCtas; b0 += 32) {
      const bool has = b0 + lane < kChunkCtas && records[b0 + lane].parts > 0;
      const unsigned all = __ballot_sync(0xffffffffu, has);
      if (has)
        list[count + __popc(all & ((1u << lane) - 1))] = b0 + lane;
      count += __popc(all);
    }
    if (lane == 0)
      listed = count;
  }
  __syncthreads();
  const int items = listed * (kRows / kCombineRows);
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const PagedRecord rec = records[list[item / (kRows / kCombineRows)]];
    const int first = item % (kRows / kCombineRows) * kCombineRows;
    // tensor row and head of slot row i
    const auto place = [&](int i, int& row, int& head) {
      const int t = i % kChunkRows;
      const int qi = rec.pair * 2 * QB + i / kChunkRows * QB + t / group;
      row = rec.row0 + qi;
      head = rec.h * group + t % group;
      return t < QB * group && qi < rec.n;
    };
    // ---- a row's maximum, sum and factor: eight threads a row
    if (tid < 8 * kCombineRows) {
      const int i = tid / 8, sub = tid % 8;
      float2 ml = make_float2(-INFINITY, 0);
      for (int p = sub; p < rec.parts; p += 8)
        merge(ml, pm[record_slot(rec, p) * kRows + first + i]);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        float2 lower = ml, upper;
        upper.x = __shfl_xor_sync(0xffffffffu, ml.x, o);
        upper.y = __shfl_xor_sync(0xffffffffu, ml.y, o);
        if (sub & o) {  // both lanes add in the same order
          const float2 t = lower;
          lower = upper;
          upper = t;
        }
        merge(lower, upper);
        ml = lower;
      }
      if (sub == 0) {
        int row, head;
        float scale = 0;
        if (place(first + i, row, head)) {
          const bool empty = ml.y == 0;
          scale = empty ? 0.0F : 1.0F / ml.y;
          if (a.gate)
            scale /= 1 + expf(-to_float(static_cast<const T*>(
                             a.gate)[size_t(row) * a.ldg + head]));
          if (a.lse)
            a.lse[size_t(row) * a.heads + head] =
                empty ? -INFINITY : (ml.x + log2f(ml.y)) * kLn2;
        }
        row_scales[i] = make_float2(ml.x, scale);
      }
    }
    __syncthreads();
    // ---- the outputs: slots lie [dim / 4][row][4] (lane = row)
    for (int d4 = warp; d4 < kQuads; d4 += kThreads / 32) {
      const int i = lane;
      const float top = row_scales[i].x;
      const size_t step = size_t(kRows) * DIM;
      const float* src = a.chunk_part + (size_t(d4) * kRows + first + i) * 4;
      float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 1
      for (int p0 = 0; p0 < rec.parts; p0 += kAhead) {
        float4 v[kAhead];
        float f[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          f[k] = 0;
          v[k] = make_float4(0, 0, 0, 0);
          if (p0 + k < rec.parts) {
            const int sl = record_slot(rec, p0 + k);
            v[k] = *reinterpret_cast<const float4*>(src + sl * step);
            f[k] = pm[sl * kRows + first + i].x;
          }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          if (p0 + k >= rec.parts)
            break;
          const float w = f[k] == -INFINITY ? 1.0F : ex2(f[k] - top);
          o.x = fmaf(v[k].x, w, o.x);
          o.y = fmaf(v[k].y, w, o.y);
          o.z = fmaf(v[k].z, w, o.z);
          o.w = fmaf(v[k].w, w, o.w);
        }
      }
      const float scale = row_scales[i].y;
      *reinterpret_cast<float4*>(&tile[i][d4 * 4]) =
          make_float4(o.x * scale, o.y * scale, o.z * scale, o.w * scale);
    }
    __syncthreads();
    for (int e = tid; e < kCombineRows * kQuads; e += kThreads) {
      const int i = e / kQuads, d4 = e % kQuads;
      int row, head;
      if (!place(first + i, row, head))
        continue;
      const float4 y = *reinterpret_cast<const float4*>(&tile[i][d4 * 4]);
      T* out = static_cast<T*>(a.out) + size_t(row) * a.ldo +
               size_t(head) * DIM + d4 * 4;
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(out) = y;
      else
        *reinterpret_cast<uint2*>(out) =
            make_uint2(pack2(y.x, y.y, T{}), pack2(y.z, y.w, T{}));
    }
    __syncthreads();
  }
}

template <typename T, int DIM>
__global__ void __launch_bounds__(512)
    paged_combine_kernel(const __grid_constant__ PagedAttentionArgs a,
                         bool decode, bool chunks) {
  allow_dependents();
  grid_dependency_wait();
  if (decode)
    combine_single<T, DIM>(a);
  if (chunks)
    combine_chunks<T, DIM>(a);
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
  const bool chunks = !paged_single(a.t.max_rows, group);
  if (chunks) {
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
                       dim3(chunks ? kChunkCtas : kDecodeCtas),
                       dim3(chunks ? 512 : 128), 0,
                       stream, true, a, group <= kDecodeMaxGroup, chunks);
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
