// Eviction by accumulated weight (lfm3_cuda_paged_evict), two kernels.
//
// select  a cluster of blocks per sequence (eight, fewer when the sequences
//         fill the GPU), each with a stretch of its rows: their weights
//         as order-preserving keys (in shared memory up to kStagedRows a
//         block, read again beyond), the (keep - recent)-th largest of those
//         before the last `recent` rows by a radix select (digits of 11, 11
//         and 10 bits; every block adds up the cluster's histograms through
//         distributed shared memory), then the kept rows' numbers in row
//         order: above the threshold, or at it while any are still due, the
//         lower rows first.
// move    kept row j of number kept[j] >= j goes to row j. Into other pages
//         the rows are independent: a warp copies whole rows. In place,
//         blocks own 16-byte columns of the rows and so order their reads and
//         writes alone: rows in batches, a batch's reads all done before its
//         writes, and no write touches what a later batch reads (kept[j] >=
//         j), so the next batch is read before the barrier, too.
// One sequence of 32000 rows of 4 heads of 128, 8192 kept: 27 us into other
// pages, most of it the selection's latency (three passes over eight SMs); 48
// us in place, where a block moves a single 16-byte column, half a sector, so
// that all SMs have one. 24 sequences of 900 to 9000 rows, 2000 kept: 55 us
// either way (26 us are the bytes: the weights once, each kept row once each
// way).
#include <cooperative_groups.h>

#include <algorithm>

#include "kernels.cuh"
#include "paged.cuh"

namespace lfm3 {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kSelectRows = 4;         // consecutive rows of a thread
constexpr int kSelectCluster = 8;
constexpr int kStagedRows = 16 * 1024;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 4;           // rows of a thread in a batch

// Order-preserving key of a weight: larger weight, larger key; -0 is 0; NaN
// is above every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w)
    return 0xffffffffu;
  const uint32_t b = __float_as_uint(w == 0 ? 0.0F : w);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ uint32_t key_at(const PagedEvictArgs& a, int s,
                                           int row) {
  const int pool = paged_row(a.t, a.t.table, s, row);
  if (pool < 0) {
    report_error(kErrPagedTable);
    return 0;
  }
  return weight_key(a.weights[pool]);
}

// Exclusive sum over the block in thread order; *total gets the whole sum.
template <typename N>
__device__ N block_scan(N v, N* warp_sums, N* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  N inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o)
      inc += t;
  }
  __syncthreads();  // earlier readers of warp_sums are done
  if (lane == 31)
    warp_sums[warp] = inc;
  __syncthreads();
  // every warp scans the 32 warps' sums
  N w = warp_sums[lane], all = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N t = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o)
      all += t;
  }
  *total = __shfl_sync(0xffffffffu, all, 31);
  return inc - v + __shfl_sync(0xffffffffu, all - w, warp);
}

__global__ void __launch_bounds__(kSelectThreads)
    paged_evict_select_kernel(const __grid_constant__ PagedEvictArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ uint32_t keys[];  // [kStagedRows]
  alignas(16) __shared__ uint32_t hist[3][kBins];
  __shared__ unsigned long long sums[kSelectThreads / 32];
  __shared__ uint32_t digit, due;
  __shared__ uint32_t totals[2];  // this block's sure rows, and at threshold
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int s = blockIdx.x / ranks, tid = threadIdx.x, lane = tid % 32;
  grid_dependency_wait();
  allow_dependents();
  int length = a.t.lengths[s];
  if (length < 0 || int64_t(length) > int64_t(a.t.table_pages) * a.t.page_rows) {
    if (tid == 0)
      report_error(kErrPagedTable);
    length = 0;  // counts as an empty sequence
  }
  const int count = min(length, a.keep);
  int* kept = a.kept + size_t(s) * a.keep;
  for (int i = tid; i < 3 * kBins; i += kSelectThreads)
    hist[0][i] = 0;
  cluster.sync();  // every thread has the length: out_lengths may be lengths
  if (tid == 0 && rank == 0)
    a.out_lengths[s] = count;
  if (length <= a.keep) {
    for (int j = rank * kSelectThreads + tid; j < count;
         j += ranks * kSelectThreads)
      kept[j] = j;
    return;
  }
  const int old = length - a.recent;         // rows that compete
  const uint32_t want = a.keep - a.recent;   // of them stay (want < old)
  // this block's rows
  const int per = (length + ranks - 1) / ranks;
  const int row0 = min(rank * per, length), row1 = min(row0 + per, length);
  const int mid = min(row1, old);  // those before it compete
  const bool staged = per <= kStagedRows;
  if (staged && want > 0) {
#pragma unroll 4
    for (int t = row0 + tid; t < mid; t += kSelectThreads)
      keys[t - row0] = key_at(a, s, t);
  }
  // (the last `recent` rows stay for sure)
  uint32_t prefix = 0, mask = 0, remaining = want;
  uint32_t own_sure = max(row1 - max(row0, old), 0), own_ties = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3 && want > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bins = pass == 2 ? 1024 : 2048;
    __syncthreads();
    for (int t0 = row0; t0 < mid; t0 += kSelectThreads) {
      const int t = t0 + tid;
      uint32_t bin = 0xffffffffu;
      if (t < mid) {
        const uint32_t key = staged ? keys[t - row0] : key_at(a, s, t);
        if ((key & mask) == prefix)
          bin = (key >> shift) & (bins - 1);
      }
      // rows of equal weight (all zero, say) count as one addition
      int same;
      __match_all_sync(0xffffffffu, bin, &same);
      if (same) {
        if (lane == 0 && bin != 0xffffffffu)
          atomicAdd(&hist[pass][bin], 32u);
      } else if (bin != 0xffffffffu) {
        atomicAdd(&hist[pass][bin], 1u);
      }
    }
    cluster.sync();
    // the bin that holds the remaining-th largest: thread i has the two bins
    // from the top that begin at 2 i. One scan carries the cluster's counts
    // and this block's own.
    const uint32_t b0 = kBins - 1 - 2 * tid;
    const uint32_t o0 = hist[pass][b0], o1 = hist[pass][b0 - 1];
    uint32_t h0 = 0, h1 = 0;
#pragma unroll
    for (int r = 0; r < kSelectCluster; ++r) {
      const uint2 h =
          r < ranks ? *reinterpret_cast<const uint2*>(cluster.map_shared_rank(
                          &hist[pass][b0 - 1], r))
                    : make_uint2(0, 0);
      h1 += h.x;
      h0 += h.y;
    }
    using Two = unsigned long long;
    Two all;
    const Two scan =
        block_scan<Two>(Two(h0 + h1) << 32 | (o0 + o1), sums, &all);
    const uint32_t above = uint32_t(scan >> 32);
    if (above < remaining && remaining <= above + h0 + h1) {
      const bool second = remaining > above + h0;
      digit = second ? b0 - 1 : b0;
      due = remaining - above - (second ? h0 : 0);
      totals[0] = uint32_t(scan) + (second ? o0 : 0);  // of this block, above
      totals[1] = second ? o1 : o0;
    }
    __syncthreads();
    prefix |= digit << shift;
    mask |= (bins - 1) << shift;
    remaining = due;
    own_sure += totals[0];
    own_ties = totals[1];
  }
  // A row stays for sure, or is at the threshold: `remaining` of those stay,
  // the lowest. Bit 2 r: sure, 2 r + 1: at the threshold, of row t0 + r.
  const auto flags_at = [&](int t0) {
    uint32_t flags = 0;
#pragma unroll
    for (int r = 0; r < kSelectRows; ++r) {
      const int t = t0 + r;
      if (t >= row1)
        continue;
      if (t >= old) {
        flags |= 1u << (2 * r);
      } else if (want > 0) {
        const uint32_t key = staged ? keys[t - row0] : key_at(a, s, t);
        flags |= (key > prefix ? 1u : key == prefix ? 2u : 0u) << (2 * r);
      }
    }
    return flags;
  };
  constexpr uint32_t kSureBits = 0x55, kTieBits = 0xAA;
  constexpr int kStep = kSelectThreads * kSelectRows;
  static_assert(kSelectRows == 4, "the masks are of four rows");
  __syncthreads();  // the last pass has read totals
  if (tid == 0) {
    totals[0] = own_sure;
    totals[1] = own_ties;
  }
  cluster.sync();
  uint32_t sure = 0, ties = 0;  // rows before this block's
#pragma unroll
  for (int r = 0; r < kSelectCluster; ++r)
    if (r < rank) {
      const uint32_t* t = cluster.map_shared_rank(totals, r);
      sure += t[0];
      ties += t[1];
    }
  for (int s0 = row0; s0 < row1; s0 += kStep) {
    const int t0 = s0 + tid * kSelectRows;
    const uint32_t flags = flags_at(t0);
    unsigned long long all;
    const uint32_t before = uint32_t(block_scan<unsigned long long>(
        __popc(flags & kSureBits) | __popc(flags & kTieBits) << 16, sums,
        &all));
    uint32_t at = sure + (before & 0xffffu), tie = ties + (before >> 16);
#pragma unroll
    for (int r = 0; r < kSelectRows; ++r) {
      const bool stays = flags >> (2 * r) & 1;
      const bool even = flags >> (2 * r + 1) & 1;
      // rows before it that stay: the sure ones and the first ties
      const uint32_t place = at + min(tie, remaining);
      if ((stays || (even && tie < remaining)) && place < uint32_t(a.keep))
        kept[place] = t0 + r;
      at += stays;
      tie += even;
    }
    sure += uint32_t(all) & 0xffffu;
    ties += uint32_t(all) >> 16;
  }
  cluster.sync();  // the others have read this block's shared memory
}

// Rows into other pages, whole: a warp a row, over the sequence's blocks.
__device__ void copy_rows(const PagedEvictArgs& a, int s, int count,
                          int row_pieces) {
  constexpr int kWarps = kMoveThreads / 32;
  const int lane = threadIdx.x % 32;
  const int* kept = a.kept + size_t(s) * a.keep;
  const int stride = gridDim.x * kWarps;
  // row numbers and page ids are read a row ahead
  int j = blockIdx.x * kWarps + threadIdx.x / 32;
  int from = -1, to = -1;
  const auto find = [&](int row, int& f, int& t) {
    f = row < count ? paged_row(a.t, a.t.table, s, kept[row]) : 0;
    t = row < count ? paged_row(a.t, a.out_table, s, row) : 0;
  };
  find(j, from, to);
  for (; j < count; j += stride) {
    int f = -1, t = -1;
    if (from < 0 || to < 0) {
      report_error(kErrPagedTable);
      find(j + stride, from, to);
      continue;
    }
    const uint4* ks = reinterpret_cast<const uint4*>(a.t.k) + size_t(from) * row_pieces;
    const uint4* vs = reinterpret_cast<const uint4*>(a.t.v) + size_t(from) * row_pieces;
    uint4* kd = reinterpret_cast<uint4*>(a.t.k) + size_t(to) * row_pieces;
    uint4* vd = reinterpret_cast<uint4*>(a.t.v) + size_t(to) * row_pieces;
    bool looked = false;
    for (int p = lane; p < row_pieces; p += 64) {
      const bool two = p + 32 < row_pieces;
      const uint4 k0 = ks[p], v0 = vs[p];
      const uint4 k1 = two ? ks[p + 32] : k0, v1 = two ? vs[p + 32] : v0;
      if (!looked)
        find(j + stride, f, t);
      looked = true;
      kd[p] = k0;
      vd[p] = v0;
      if (two) {
        kd[p + 32] = k1;
        vd[p + 32] = v1;
      }
    }
    if (!looked)
      find(j + stride, f, t);
    if (lane == 0)
      a.weights[to] = a.weights[from];
    from = f;
    to = t;
  }
}

// Block (slice, sequence). In place: 16-byte columns [slice * cols, + cols) of
// the rows of K, then V; block `slices` moves the weights.
__global__ void __launch_bounds__(kMoveThreads, 3)
    paged_evict_move_kernel(const __grid_constant__ PagedEvictArgs a,
                            int row_pieces, int cols, int slices) {
  const int s = blockIdx.y, tid = threadIdx.x;
  grid_dependency_wait();
  allow_dependents();
  const int count = a.out_lengths[s];  // the select kernel's, <= keep
  const int* kept = a.kept + size_t(s) * a.keep;
  if (count == 0)
    return;
  if (a.out_table[size_t(s) * a.t.table_stride] !=
      a.t.table[size_t(s) * a.t.table_stride]) {
    copy_rows(a, s, count, row_pieces);
    return;
  }
  if (blockIdx.x > slices)
    return;
  const bool weights = blockIdx.x == slices;
  const int c = weights ? 1 : cols;
  const int piece = blockIdx.x * cols + tid % c;
  const bool mine = weights || piece < 2 * row_pieces;
  uint4* pool = reinterpret_cast<uint4*>(piece < row_pieces ? a.t.k : a.t.v);
  const int col = piece < row_pieces ? piece : piece - row_pieces;
  const int step = kMoveThreads / c;  // rows between a thread's rows
  const int batch = step * kMoveRows;
  struct Rows {
    int from[kMoveRows], to[kMoveRows];
  };
  const auto find = [&](int j0, Rows& r) {
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      const int j = j0 + k * step + tid / c;
      r.from[k] = r.to[k] = -1;
      if (j < count && mine) {
        r.from[k] = paged_row(a.t, a.t.table, s, kept[j]);
        r.to[k] = paged_row(a.t, a.out_table, s, j);
        if (r.from[k] < 0 || r.to[k] < 0) {
          report_error(kErrPagedTable);
          r.from[k] = r.to[k] = -1;
        }
        if (r.from[k] == r.to[k])
          r.from[k] = r.to[k] = -1;  // already there
      }
    }
  };
  const auto read = [&](const Rows& r, uint4(&data)[kMoveRows]) {
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k)
      if (r.from[k] >= 0) {
        if (weights)
          data[k].x = __float_as_uint(a.weights[r.from[k]]);
        else
          data[k] = pool[size_t(r.from[k]) * row_pieces + col];
      }
  };
  Rows now, next;
  uint4 data[kMoveRows], ahead[kMoveRows];
  find(0, now);
  read(now, data);
  find(batch, next);
  for (int j0 = 0; j0 < count; j0 += batch) {
    read(next, ahead);
    Rows later;
    find(j0 + 2 * batch, later);
    __syncthreads();  // the batch is read before any of it is written
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k)
      if (now.to[k] >= 0) {
        if (weights)
          a.weights[now.to[k]] = __uint_as_float(data[k].x);
        else
          pool[size_t(now.to[k]) * row_pieces + col] = data[k];
      }
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k)
      data[k] = ahead[k];
    now = next;
    next = later;
  }
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvictArgs& a, int dim,
                               cudaStream_t stream) {
  cudaError_t e = ensure_dynamic_smem(
      reinterpret_cast<const void*>(paged_evict_select_kernel),
      kStagedRows * 4);
  if (e != cudaSuccess)
    return e;
  int cluster = kSelectCluster;
  while (cluster > 1 && a.t.sequences * cluster > 148)
    cluster /= 2;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(a.t.sequences * cluster));
  config.blockDim = dim3(kSelectThreads);
  config.dynamicSmemBytes = kStagedRows * 4;
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {unsigned(cluster), 1, 1};
  config.attrs = attr;
  config.numAttrs = 2;
  note_launch();
  if ((e = cudaLaunchKernelEx(&config, paged_evict_select_kernel, a)))
    return e;
  const int pieces = a.t.kv_heads * dim / 8;  // 16-byte pieces of a row
  // In place, columns of a block: as many (up to 8, 128 bytes) as leave a
  // block for every SM. Whole rows want 16 warps of an SM.
  int cols = 8;
  while (cols > 1 && (2 * pieces + cols - 1) / cols * a.t.sequences < 148)
    cols /= 2;
  const int slices = (2 * pieces + cols - 1) / cols;
  const int blocks =
      std::max(slices + 1, (148 * 2 + a.t.sequences - 1) / a.t.sequences);
  return launch_kernel(paged_evict_move_kernel, dim3(blocks, a.t.sequences),
                       dim3(kMoveThreads), 0, stream, true, a, pieces, cols,
                       slices);
}

}  // namespace lfm3
