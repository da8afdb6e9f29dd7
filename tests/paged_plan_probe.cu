// Runs the paged kernels' plans on device tables alone, without tensors: one
// warp a block, as many blocks as the kernels have. For tests.
#include "../lfm3-gufo-extension_b200/csrc/paged_plan.cuh"

namespace {

using namespace lfm3;

// out: share, places of the line, units that the blocks' segments hold,
// stretches begun, segments
using Out = unsigned long long;

__global__ void chunks(PagedTables t, int group, int window, int extra,
                       bool walk, Out* out) {
  PagedLine<ChunkUnits> line(t, ChunkUnits{group, window, 1, extra});
  const int64_t share = chunk_plan(line);
  const int64_t total = line.total * t.kv_heads;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    out[0] = share;
    out[1] = total;
  }
  const int64_t end = min(share * (blockIdx.x + 1), total);
  ChunkSegment g;
  for (int64_t at = share * blockIdx.x;
       walk && chunk_segment(line, at, end, g); at += g.units)
    if (threadIdx.x == 0) {
      atomicAdd(&out[2], Out(g.count));
      atomicAdd(&out[3], Out(g.u0 == 0));
      atomicAdd(&out[4], 1ull);
    }
}

__global__ void weights(PagedTables t, int group, int window, bool walk,
                        Out* out) {
  PagedLine line(t, WeightUnits{group, window});
  const int64_t total = line.total * t.kv_heads;
  const int64_t share = paged_share(total, kWeightCtas, 1);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    out[0] = share;
    out[1] = total;
  }
  const int64_t end = min(share * (blockIdx.x + 1), total);
  WeightSegment g;
  for (int64_t at = share * blockIdx.x;
       walk && weight_segment(line, group, window, at, end, g); at += g.count)
    if (threadIdx.x == 0) {
      atomicAdd(&out[2], Out(g.count));
      atomicAdd(&out[3], Out(g.u0 == 0));
      atomicAdd(&out[4], 1ull);
    }
}

__global__ void decode(PagedTables t, int group, int window, Out* out) {
  const DecodePlan plan = decode_plan(t, group, window);
  PagedLine line(t, DecodeUnits{group, window, plan.pad, plan.extra});
  if (threadIdx.x == 0) {
    out[0] = plan.share;
    out[1] = line.total * t.kv_heads;
  }
}

}  // namespace

// what: 0 chunks, 1 key weights, 2 single tokens. starts, lengths and out are
// device arrays; out has five zeros.
extern "C" int paged_plan_probe(int what, const int* starts, const int* lengths,
                                int sequences, int kv_heads, int group,
                                int window, int extra, int walk, int table_pages,
                                int page_rows, int rows, int max_rows,
                                unsigned long long* out) {
  PagedTables t{};
  t.starts = starts;
  t.lengths = lengths;
  t.sequences = sequences;
  t.kv_heads = kv_heads;
  t.table_pages = table_pages;
  t.page_rows = page_rows;
  t.rows = rows;
  t.max_rows = max_rows;
  if (what == 0)
    chunks<<<kChunkCtas, 32>>>(t, group, window, extra, walk, out);
  else if (what == 1)
    weights<<<kWeightCtas, 32>>>(t, group, window, walk, out);
  else
    decode<<<1, 32>>>(t, group, window, out);
  return int(cudaDeviceSynchronize());
}
