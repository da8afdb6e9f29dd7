// Paged K/V cache operators (lfm3_cuda_paged_*): the descriptors as the
// kernels see them, the rules every kernel reads the device tables by, and
// the launch entry points.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/lfm3_cuda.h"
#include "common.cuh"

namespace lfm3 {

constexpr int kMaxPagedSequences = 4096;
constexpr int kMaxPagedGroup = 128;

// The device arrays of lfm3_paged_cache and lfm3_paged_batch, by value.
struct PagedTables {
  __half* k;
  __half* v;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;
  int pages, page_rows, kv_heads, sequences, table_pages, table_stride;
  int rows, max_rows;
};

// A sequence of the batch: its new rows are tensor rows row0 .. row0 + n - 1
// and the last n of its `length` cached rows.
struct PagedSequence {
  int row0, n, length;
  bool broken;
};

// The rule on starts and lengths (the host check and every kernel): a
// sequence whose entries are broken takes part with no rows, or no keys.
__host__ __device__ inline PagedSequence paged_sequence(const PagedTables& t,
                                                        int s) {
  const int begin = t.starts[s], end = t.starts[s + 1], length = t.lengths[s];
  PagedSequence q{begin, 0, 0, false};
  if (begin < 0 || end < begin || end > t.rows || end - begin > t.max_rows)
    q.broken = true;
  else
    q.n = end - begin;
  if (length < 0 ||
      int64_t(length) > int64_t(t.table_pages) * t.page_rows)
    q.broken = true;
  else
    q.length = length;
  return q;
}

// Pool row (0 .. pages * page_rows - 1) of row `row` of sequence s, or -1
// where the page id is outside the pool. row must be inside the sequence.
__host__ __device__ inline int paged_row(const PagedTables& t,
                                         const int32_t* table, int s, int row) {
  const int slot = row / t.page_rows;
  const int page = table[size_t(s) * t.table_stride + slot];
  return page < 0 || page >= t.pages
             ? -1
             : page * t.page_rows + (row - slot * t.page_rows);
}

// Element types of q, k, v, out and gate.
template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_float(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_float(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) {
  return __float2bfloat16_rn(v);
}

// Two FP32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\n"
      "mov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\n"
      "mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\n"
      "add.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// The elements of 16 bytes, and back (one rounding).
__device__ __forceinline__ void unpack16(uint4 u, float (&x)[4], float) {
  x[0] = __uint_as_float(u.x);
  x[1] = __uint_as_float(u.y);
  x[2] = __uint_as_float(u.z);
  x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack16(uint4 u, float (&x)[8], __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack16(uint4 u, float (&x)[8],
                                         __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 pack16(const float (&x)[4], float) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]),
                    __float_as_uint(x[2]), __float_as_uint(x[3]));
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&x)[8], T t) {
  return make_uint4(pack2(x[0], x[1], t), pack2(x[2], x[3], t),
                    pack2(x[4], x[5], t), pack2(x[6], x[7], t));
}

// Pairs of FP32 values in 64-bit registers.
using F32x2 = unsigned long long;
__device__ __forceinline__ F32x2 pair(float a, float b) {
  F32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 both(F32x2 a) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
  return d;
}
__device__ __forceinline__ F32x2 fma_pair(F32x2 a, F32x2 b, F32x2 c) {
  F32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ F32x2 mul_pair(F32x2 a, F32x2 b) {
  F32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

struct PagedHeadsArgs {
  PagedTables t;
  const int32_t* positions;
  const void *q, *k, *v;
  void* q_out;
  size_t ldq, ldk, ldv, ldo;
  const float *q_norm, *k_norm, *freq, *factors;
  int heads;
  float eps;
};
cudaError_t launch_paged_heads(const PagedHeadsArgs& a, uint32_t type, int dim,
                               cudaStream_t stream);

struct PagedAttentionArgs {
  // [slab of 64 dims][pool row][64], boxes of 16 rows and a whole head
  alignas(64) CUtensorMap kmap16;
  alignas(64) CUtensorMap vmap16;
  // the same pools, boxes of box_rows rows of one slab
  alignas(64) CUtensorMap kmap;
  alignas(64) CUtensorMap vmap;
  int box_rows;
  PagedTables t;
  const void* q;
  const void* gate;
  void* out;
  float* lse;
  size_t ldq, ldg, ldo;
  int heads, window;
  // slots of [group][dim] outputs, then of (max, sum), then the records
  float* decode_part;
  // slots of [dim / 4][256 rows][4], then of (max, sum), then the records
  float* chunk_part;
  void* workspace;
};
// Single-token sequences of the batch, and the slots' floats.
cudaError_t launch_paged_decode(const PagedAttentionArgs& a, uint32_t type,
                                int dim, cudaStream_t stream);
size_t paged_decode_floats(int dim, int group);
// The other sequences (chunks, and wide groups), and the slots' floats.
cudaError_t launch_paged_chunk(const PagedAttentionArgs& a, uint32_t type,
                               int dim, cudaStream_t stream);
size_t paged_chunk_floats(int dim);
size_t paged_attention_workspace(const PagedTables& t, int dim, int heads);
cudaError_t launch_paged_attention(const PagedAttentionArgs& a, uint32_t type,
                                   int dim, cudaStream_t stream);

struct PagedKeyWeightsArgs {
  alignas(64) CUtensorMap kmap;  // keys, boxes of box_rows rows of one slab
  // the queries' fp16 terms, boxes of one query or a whole column block
  alignas(64) CUtensorMap qmap1[2];
  alignas(64) CUtensorMap qmap[2];
  int box_rows;
  PagedTables t;
  const void* q;
  const float* lse;
  float* weights;
  size_t ldq;
  int heads, window;
  void* workspace;
  __half* terms;    // [term][rows][heads][dim]
  float2* factors;  // [rows][heads]: score factor, lse in base 2
  float* part;      // slots of 256 sums, then the records
};
size_t paged_key_weights_workspace(const PagedTables& t, int dim, int heads);
cudaError_t launch_paged_key_weights(const PagedKeyWeightsArgs& a,
                                     uint32_t type, int dim,
                                     cudaStream_t stream);

struct PagedEvictArgs {
  PagedTables t;
  const int32_t* out_table;
  int32_t* out_lengths;
  float* weights;
  int32_t* kept;
  int keep, recent;
};
cudaError_t launch_paged_evict(const PagedEvictArgs& a, int dim,
                               cudaStream_t stream);

}  // namespace lfm3
