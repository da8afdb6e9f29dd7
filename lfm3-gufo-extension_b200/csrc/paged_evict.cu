// Eviction by accumulated weight (lfm3_cuda_paged_evict).
//
// select  one block per sequence: the (keep - recent)-th largest weight among
//         the rows before the last `recent` by a 4-pass radix select on
//         order-preserving keys (8 bits a pass), then one pass in row order
//         that writes the kept rows' numbers (above the threshold, or at it
//         while any are still due: the lower rows first).
// move    kept row j of number kept[j] >= j goes to row j. Blocks own column
//         slices, so a block alone orders its reads and writes: it moves rows
//         in order, a batch's reads all done before its writes, and no later
//         batch reads what an earlier one wrote (kept[j] >= j). That makes
//         the move safe in place.
#include "kernels.cuh"
#include "paged.cuh"

namespace lfm3 {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kMoveThreads = 256;

// Order-preserving key of a weight: larger weight, larger key; -0 is 0; NaN
// is above every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w)
    return 0xffffffffu;
  const uint32_t b = __float_as_uint(w == 0 ? 0.0F : w);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A length outside the table counts as an empty sequence.
__device__ __forceinline__ int evict_length(const PagedTables& t, int s,
                                            bool& broken) {
  const int length = t.lengths[s];
  broken = length < 0 || int64_t(length) > int64_t(t.table_pages) * t.page_rows;
  return broken ? 0 : length;
}

__device__ __forceinline__ float weight_at(const PagedEvictArgs& a, int s,
                                           int row) {
  const int pool = paged_row(a.t, a.t.table, s, row);
  if (pool < 0) {
    report_error(kErrPagedTable);
    return 0;
  }
  return a.weights[pool];
}

// Exclusive sum over the block in thread order; *total gets the whole sum.
__device__ int block_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o)
      inc += t;
  }
  __syncthreads();
  if (lane == 31)
    warp_sums[warp] = inc;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    before += w < warp ? warp_sums[w] : 0;
    all += warp_sums[w];
  }
  *total = all;
  return before + inc - v;
}

__global__ void __launch_bounds__(kSelectThreads)
    paged_evict_select_kernel(const __grid_constant__ PagedEvictArgs a) {
  __shared__ unsigned hist[256];
  __shared__ int sums[kSelectThreads / 32];
  __shared__ unsigned digit, due;
  const int s = blockIdx.x, tid = threadIdx.x;
  bool broken;
  const int length = evict_length(a.t, s, broken);
  if (broken && tid == 0)
    report_error(kErrPagedTable);
  int* kept = a.kept + size_t(s) * a.keep;
  const int count = min(length, a.keep);
  // every thread has the length: out_lengths may be the same array
  __syncthreads();
  if (tid == 0)
    a.out_lengths[s] = count;
  if (length <= a.keep) {
    for (int j = tid; j < count; j += kSelectThreads)
      kept[j] = j;
    return;
  }
  const int old = length - a.recent;   // rows that compete
  const int want = a.keep - a.recent;  // of them stay (want < old)
  uint32_t prefix = 0, mask = 0;
  unsigned remaining = want;
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelectThreads)
        hist[i] = 0;
      __syncthreads();
      for (int t = tid; t < old; t += kSelectThreads) {
        const uint32_t key = weight_key(weight_at(a, s, t));
        if ((key & mask) == prefix)
          atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        unsigned left = remaining;
        int b = 255;
        while (b > 0 && hist[b] < left)
          left -= hist[b--];
        digit = b;
        due = left;
      }
      __syncthreads();
      prefix |= digit << shift;
      mask |= 255u << shift;
      remaining = due;
      __syncthreads();
    }
  }
  // `remaining` rows at the threshold stay, the lowest first
  int out = 0, ties = 0;
  for (int t0 = 0; t0 < length; t0 += kSelectThreads) {
    const int t = t0 + tid;
    bool keep = false, tie = false;
    if (t < length) {
      if (t >= old)
        keep = true;
      else if (want > 0) {
        const uint32_t key = weight_key(weight_at(a, s, t));
        keep = key > prefix;
        tie = key == prefix;
      }
    }
    int all;
    const int rank = ties + block_scan(tie, sums, &all);
    ties += all;
    if (tie && rank < int(remaining))
      keep = true;
    const int at = out + block_scan(keep, sums, &all);
    out += all;
    if (keep && at < a.keep)
      kept[at] = t;
  }
}

// Block (slice, sequence): 16-byte columns [slice * cols, +cols) of K's then
// V's rows; the last slice moves the weights.
__global__ void __launch_bounds__(kMoveThreads)
    paged_evict_move_kernel(const __grid_constant__ PagedEvictArgs a,
                            int row_pieces, int cols) {
  const int s = blockIdx.y, tid = threadIdx.x;
  const int count = a.out_lengths[s];  // the select kernel's, <= keep
  const int* kept = a.kept + size_t(s) * a.keep;
  const bool weights = blockIdx.x == gridDim.x - 1;
  const int piece = blockIdx.x * cols + tid % cols;
  const int per = kMoveThreads / cols;  // rows of a batch
  const bool is_v = piece >= row_pieces;
  uint4* pool = reinterpret_cast<uint4*>(is_v ? a.t.v : a.t.k);
  const int col = is_v ? piece - row_pieces : piece;
  const bool mine = !weights && piece < 2 * row_pieces;
  for (int j0 = 0; j0 < count; j0 += weights ? kMoveThreads : per) {
    const int j = j0 + (weights ? tid : tid / cols);
    int from = -1, to = -1;
    if (j < count && (weights || mine)) {
      from = paged_row(a.t, a.t.table, s, kept[j]);
      to = paged_row(a.t, a.out_table, s, j);
      if (from < 0 || to < 0) {
        report_error(kErrPagedTable);
        from = to = -1;
      }
    }
    uint4 data = make_uint4(0, 0, 0, 0);
    float w = 0;
    if (from >= 0) {
      if (weights)
        w = a.weights[from];
      else
        data = pool[size_t(from) * row_pieces + col];
    }
    __syncthreads();  // the batch is read before any of it is written
    if (to >= 0) {
      if (weights)
        a.weights[to] = w;
      else
        pool[size_t(to) * row_pieces + col] = data;
    }
  }
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvictArgs& a, int dim,
                               cudaStream_t stream) {
  if (cudaError_t e = launch_kernel(paged_evict_select_kernel,
                                    dim3(a.t.sequences), dim3(kSelectThreads),
                                    0, stream, false, a))
    return e;
  const int pieces = a.t.kv_heads * dim / 8;  // 16-byte pieces of a row
  const int cols = 4;
  return launch_kernel(paged_evict_move_kernel,
                       dim3((2 * pieces + cols - 1) / cols + 1, a.t.sequences),
                       dim3(kMoveThreads), 0, stream, false, a, pieces, cols);
}

}  // namespace lfm3
