// extern "C" entry points of the paged K/V cache operators: argument checks
// (before any CUDA call), then one launcher each.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <memory>
#include <new>

#include "../../include/lfm3_cuda.h"
#include "kernels.cuh"
#include "paged.cuh"

namespace {

using lfm3::PagedTables;

int Invalid(const char* message) {
  return lfm3::set_last_error(LFM3_ERR_INVALID, message);
}
int Unsupported(const char* message) {
  return lfm3::set_last_error(LFM3_ERR_UNSUPPORTED, message);
}
// A launcher's status. A failed launch also sets the runtime's last error,
// which the caller's own next check would take for its own: cleared here.
int Status(cudaError_t e) {
  if (e == cudaSuccess)
    return LFM3_OK;
  cudaGetLastError();
  return lfm3::set_last_error(LFM3_ERR_CUDA, cudaGetErrorString(e));
}
bool Aligned16(const void* p) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0;
}
// Kernels read and write arrays an element at a time at least: each has to be
// aligned to its elements (a misaligned access would end the context). NULL is.
bool Aligned(size_t bytes, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (reinterpret_cast<uintptr_t>(p) % bytes)
      return false;
  return true;
}

// The descriptors' own numbers and pointers. dim and kv_heads first: the
// other operators answer UNSUPPORTED for shapes, whatever the pointers are.
int CheckCache(const lfm3_paged_cache* c) {
  if (!c)
    return Invalid("paged cache descriptor is NULL");
  if (c->dim != 64 && c->dim != 128)
    return Unsupported("paged cache: dim must be 64 or 128");
  if (c->kv_heads < 1 || c->kv_heads > 1024)
    return Unsupported("paged cache: kv_heads must be 1..1024");
  if (c->page_rows < 16 || c->page_rows % 16)
    return Unsupported("paged cache: page_rows must be a multiple of 16");
  if (c->sequences < 0 || c->sequences > lfm3::kMaxPagedSequences)
    return Unsupported("paged cache: sequences must be 0..4096");
  if (c->pages < 1 || c->table_pages < 1 || c->table_stride < c->table_pages)
    return Invalid("paged cache: pages, table_pages and table_stride");
  // TMA row coordinates and row numbers (rounded up to tiles) are 32-bit;
  // products are 64-bit
  if (int64_t(c->pages) * c->page_rows > INT_MAX - 4096 ||
      int64_t(c->table_pages) * c->page_rows > INT_MAX - 4096)
    return Unsupported("paged cache: more than 2^31 - 4097 rows");
  if (!c->k || !c->v || !c->table || !c->lengths)
    return Invalid("paged cache: NULL array");
  if (!Aligned16(c->k) || !Aligned16(c->v))
    return Invalid("paged cache: k and v must be 16-byte aligned");
  if (!Aligned(4, {c->table, c->lengths}))
    return Invalid("paged cache: table or lengths are not aligned");
  return LFM3_OK;
}
int CheckBatch(const lfm3_paged_batch* b) {
  if (!b)
    return Invalid("paged batch descriptor is NULL");
  if (!b->starts || b->rows < 0 || b->max_rows < 0)
    return Invalid("paged batch: starts, rows and max_rows");
  if (!Aligned(4, {b->starts}))
    return Invalid("paged batch: starts are not aligned");
  return LFM3_OK;
}
int CheckType(uint32_t type) {
  return type == LFM3_F32 || type == LFM3_F16 || type == LFM3_BF16
             ? LFM3_OK
             : Unsupported("paged operators take F32, F16 or BF16 rows");
}
int CheckHeads(int heads, const lfm3_paged_cache* c) {
  if (heads < 1 || heads % c->kv_heads ||
      heads / c->kv_heads > lfm3::kMaxPagedGroup)
    return Unsupported("paged operators: heads / kv_heads must be a whole "
                       "number up to 128");
  return LFM3_OK;
}
int CheckRows(const void* p, size_t stride, size_t width, const char* what) {
  if (!p || !Aligned16(p) || stride % 8 || stride < width ||
      stride > size_t(1) << 40)
    return Invalid(what);
  return LFM3_OK;
}
// `rows` rows of `width` elements, `stride` elements apart.
struct Rows {
  const void* p;
  size_t stride, width;
};
// Whether a row of a and a row of b have a byte in common (columns of one
// buffer do not, though their ranges overlap).
bool Overlap(const Rows& a, const Rows& b, int rows, uint32_t type) {
  using Wide = __int128;
  const size_t size = type == LFM3_F32 ? 4 : 2;
  const Wide a0 = reinterpret_cast<uintptr_t>(a.p), aw = a.width * size;
  const Wide b0 = reinterpret_cast<uintptr_t>(b.p), bw = b.width * size;
  const Wide as = Wide(a.stride) * size, bs = Wide(b.stride) * size;
  if (a0 + (rows - 1) * as + aw <= b0 || b0 + (rows - 1) * bs + bw <= a0)
    return false;
  // in the order of addresses: the row that ends first meets no later one
  for (Wide i = 0, j = 0; i < rows && j < rows;) {
    const Wide x = a0 + i * as, y = b0 + j * bs;
    if (x + aw > y && y + bw > x)
      return true;
    // rows that end before the other's begin, all at once
    if (x + aw <= y)
      i += std::max<Wide>((y - x - aw) / as, 1);
    else
      j += std::max<Wide>((x - y - bw) / bs, 1);
    // equal strides: what holds for one pair of neighbours holds for all
    if (as == bs && i > 0 && j > 0)
      return false;
  }
  return false;
}
// The caller's memory has to be of the current device, where the kernels run:
// pools, queries, their outputs and workspaces in its own or managed memory,
// the other arrays (`small`) may be pinned host memory, too. Pageable memory
// and another device's would end the context.
// The driver is asked for three attributes at once: 34 ns an array, where
// cudaPointerGetAttributes takes 58 (a call has up to 14).
struct Memory {
  int device = -1;
  int status = LFM3_OK;
  int check(const void* p, bool small, const char* what) {
    if (status != LFM3_OK || !p)
      return status;
    cudaError_t e = device < 0 ? cudaGetDevice(&device) : cudaSuccess;
    if (e != cudaSuccess)
      return status = Status(e);
    static const auto get = [] {
      void* f = nullptr;
      cudaDriverEntryPointQueryResult found;
      if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &f,
                                  cudaEnableDefault, &found) != cudaSuccess ||
          found != cudaDriverEntryPointSuccess)
        f = nullptr;
      return reinterpret_cast<decltype(&cuPointerGetAttributes)>(f);
    }();
    CUpointer_attribute names[3] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE,
                                    CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL,
                                    CU_POINTER_ATTRIBUTE_IS_MANAGED};
    unsigned type = 0;  // of memory the driver knows nothing of
    int owner = -1;
    unsigned managed = 0;  // (the driver may write one byte of it, or four)
    void* values[3] = {&type, &owner, &managed};
    if (!get || get(3, names, values, reinterpret_cast<CUdeviceptr>(p)))
      return status = Status(cudaErrorNotSupported);
    if (managed || (type == CU_MEMORYTYPE_DEVICE && owner == device) ||
        (type == CU_MEMORYTYPE_HOST && small))
      return LFM3_OK;
    return status = Invalid(what);
  }
  // (what an operator does not read is not looked at: key weights need no
  // values, heads alone read positions)
  int check(const lfm3_paged_cache* c, bool values = true) {
    constexpr const char* what = "paged cache is not on the current device";
    check(c->k, false, what);
    if (values)
      check(c->v, false, what);
    check(c->table, true, what);
    return check(c->lengths, true, what);
  }
  int check(const lfm3_paged_batch* b) {
    return check(b->starts, true, "paged batch is not on the current device");
  }
  int check(std::initializer_list<const void*> arrays, const char* what) {
    for (const void* p : arrays)
      check(p, true, what);
    return status;
  }
};

PagedTables Tables(const lfm3_paged_cache* c, const lfm3_paged_batch* b) {
  PagedTables t{};
  t.k = reinterpret_cast<__half*>(c->k);
  t.v = reinterpret_cast<__half*>(c->v);
  t.table = c->table;
  t.lengths = c->lengths;
  t.pages = c->pages;
  t.page_rows = c->page_rows;
  t.kv_heads = c->kv_heads;
  t.sequences = c->sequences;
  t.table_pages = c->table_pages;
  t.table_stride = c->table_stride;
  if (b) {
    t.starts = b->starts;
    t.rows = b->rows;
    t.max_rows = b->max_rows;
  }
  return t;
}

}  // namespace

#define CHECK(x)           \
  do {                     \
    if (const int e = (x)) \
      return e;            \
  } while (0)

extern "C" {

int lfm3_paged_check(const lfm3_paged_cache* cache,
                     const lfm3_paged_batch* batch, int shared) {
  CHECK(CheckCache(cache));
  CHECK(CheckBatch(batch));
  const PagedTables t = Tables(cache, batch);
  std::unique_ptr<bool[]> held(shared ? nullptr
                                      : new (std::nothrow) bool[t.pages]());
  if (!shared && !held)
    return Invalid("paged check: out of memory");
  char message[128];
  for (int s = 0; s < t.sequences; ++s) {
    const lfm3::PagedSequence q = lfm3::paged_sequence(t, s);
    if (q.broken) {
      snprintf(message, sizeof message,
               "paged sequence %d: starts %d..%d, length %d", s, t.starts[s],
               t.starts[s + 1], t.lengths[s]);
      return Invalid(message);
    }
    for (int64_t row = 0; row < q.length; row += t.page_rows) {
      const int pool = lfm3::paged_row(t, t.table, s, int(row));
      const bool twice = pool >= 0 && !shared && held[pool / t.page_rows];
      if (pool < 0 || twice) {
        snprintf(message, sizeof message, "paged sequence %d: page of row %d%s",
                 s, int(row), twice ? " is held already" : "");
        return Invalid(message);
      }
      if (!shared)
        held[pool / t.page_rows] = true;
    }
  }
  return LFM3_OK;
}

int lfm3_cuda_paged_heads(const lfm3_paged_cache* cache,
                          const lfm3_paged_batch* batch, uint32_t type,
                          const void* q, size_t q_stride, const void* k,
                          size_t k_stride, const void* v, size_t v_stride,
                          void* q_out, size_t q_out_stride, int heads,
                          const float* q_norm, const float* k_norm,
                          const float* frequencies, const float* factors,
                          float eps, void* stream) {
  CHECK(CheckCache(cache));
  CHECK(CheckBatch(batch));
  CHECK(CheckType(type));
  CHECK(CheckHeads(heads, cache));
  if (!frequencies || !(eps >= 0) || !std::isfinite(eps))
    return Invalid("paged heads: frequencies and eps");
  if (!Aligned(4, {batch->positions, q_norm, k_norm, frequencies, factors}))
    return Invalid("paged heads: positions, norms, frequencies or factors are "
                   "not aligned");
  if (batch->rows == 0 || cache->sequences == 0 || batch->max_rows == 0)
    return LFM3_OK;
  const size_t width = size_t(heads) * cache->dim;
  const size_t kv = size_t(cache->kv_heads) * cache->dim;
  CHECK(CheckRows(q, q_stride, width, "paged heads: q or its stride"));
  CHECK(CheckRows(k, k_stride, kv, "paged heads: k or its stride"));
  CHECK(CheckRows(v, v_stride, kv, "paged heads: v or its stride"));
  CHECK(CheckRows(q_out, q_out_stride, width,
                  "paged heads: q_out or its stride"));
  if (q_out == q && q_out_stride != q_stride)
    return Invalid("paged heads: q_out is q with another stride");
  const Rows to{q_out, q_out_stride, width};
  if ((q_out != q && Overlap(to, {q, q_stride, width}, batch->rows, type)) ||
      Overlap(to, {k, k_stride, kv}, batch->rows, type) ||
      Overlap(to, {v, v_stride, kv}, batch->rows, type))
    return Invalid("paged heads: q_out overlaps q, k or v");
  Memory memory;
  CHECK(memory.check(cache));
  CHECK(memory.check(batch));
  CHECK(memory.check(q, false, "paged heads: q is not on the current device"));
  CHECK(memory.check(q_out, false,
                     "paged heads: q_out is not on the current device"));
  CHECK(memory.check({k, v}, "paged heads: k or v is not on the current "
                             "device"));
  CHECK(memory.check({batch->positions, q_norm, k_norm, frequencies, factors},
                     "paged heads: positions, norms, frequencies or factors "
                     "are not on the current device"));
  lfm3::PagedHeadsArgs a{};
  a.t = Tables(cache, batch);
  a.positions = batch->positions;
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.ldq = q_stride, a.ldk = k_stride, a.ldv = v_stride, a.ldo = q_out_stride;
  a.q_norm = q_norm, a.k_norm = k_norm;
  a.freq = frequencies, a.factors = factors;
  a.heads = heads;
  a.eps = eps;
  return Status(lfm3::launch_paged_heads(a, type, cache->dim,
                                         static_cast<cudaStream_t>(stream)));
}

size_t lfm3_cuda_paged_attention_workspace_bytes(const lfm3_paged_cache* cache,
                                                 const lfm3_paged_batch* batch,
                                                 int heads) {
  if (CheckCache(cache) || CheckBatch(batch) || CheckHeads(heads, cache))
    return 0;
  return lfm3::paged_attention_workspace(Tables(cache, batch), cache->dim,
                                         heads);
}

int lfm3_cuda_paged_attention(const lfm3_paged_cache* cache,
                              const lfm3_paged_batch* batch, uint32_t type,
                              const void* q, size_t q_stride, const void* gate,
                              size_t gate_stride, void* out, size_t out_stride,
                              float* lse, int heads, int window,
                              void* workspace, size_t workspace_bytes,
                              void* stream) {
  CHECK(CheckCache(cache));
  CHECK(CheckBatch(batch));
  CHECK(CheckType(type));
  CHECK(CheckHeads(heads, cache));
  if (window < 0)
    return Invalid("paged attention: window must not be negative");
  if (batch->rows == 0 || cache->sequences == 0 || batch->max_rows == 0)
    return LFM3_OK;
  const size_t width = size_t(heads) * cache->dim;
  CHECK(CheckRows(q, q_stride, width, "paged attention: q or its stride"));
  CHECK(CheckRows(out, out_stride, width,
                  "paged attention: out or its stride"));
  if (out == q)
    return Invalid("paged attention: out may not be q");
  if (Overlap({out, out_stride, width}, {q, q_stride, width}, batch->rows,
              type))
    return Invalid("paged attention: out overlaps q");
  if (gate && (gate_stride < size_t(heads) || gate_stride > size_t(1) << 40))
    return Invalid("paged attention: gate stride");
  if (!Aligned(type == LFM3_F32 ? 4 : 2, {gate}) || !Aligned(4, {lse}))
    return Invalid("paged attention: gate or lse are not aligned");
  const PagedTables t = Tables(cache, batch);
  const size_t need = lfm3::paged_attention_workspace(t, cache->dim, heads);
  if (workspace_bytes < need || (need && !workspace) ||
      reinterpret_cast<uintptr_t>(workspace) % 256)
    return Invalid("paged attention: workspace too small or not 256-byte "
                   "aligned");
  Memory memory;
  CHECK(memory.check(cache));
  CHECK(memory.check(batch));
  CHECK(memory.check(q, false,
                     "paged attention: q is not on the current device"));
  CHECK(memory.check(out, false,
                     "paged attention: out is not on the current device"));
  if (need)
    CHECK(memory.check(workspace, false, "paged attention: workspace is not on "
                                         "the current device"));
  CHECK(memory.check({gate, lse}, "paged attention: gate or lse is not on the "
                                  "current device"));
  lfm3::PagedAttentionArgs a{};
  a.t = t;
  a.q = q, a.gate = gate, a.out = out, a.lse = lse;
  a.ldq = q_stride, a.ldg = gate_stride, a.ldo = out_stride;
  a.heads = heads;
  a.window = window;
  a.workspace = workspace;
  return Status(lfm3::launch_paged_attention(
      a, type, cache->dim, static_cast<cudaStream_t>(stream)));
}

size_t lfm3_cuda_paged_key_weights_workspace_bytes(
    const lfm3_paged_cache* cache, const lfm3_paged_batch* batch, int heads) {
  if (CheckCache(cache) || CheckBatch(batch) || CheckHeads(heads, cache))
    return 0;
  return lfm3::paged_key_weights_workspace(Tables(cache, batch), cache->dim,
                                           heads);
}

int lfm3_cuda_paged_key_weights(const lfm3_paged_cache* cache,
                                const lfm3_paged_batch* batch, uint32_t type,
                                const void* q, size_t q_stride,
                                const float* lse, float* weights, int heads,
                                int window, void* workspace,
                                size_t workspace_bytes, void* stream) {
  CHECK(CheckCache(cache));
  CHECK(CheckBatch(batch));
  CHECK(CheckType(type));
  CHECK(CheckHeads(heads, cache));
  if (window < 0)
    return Invalid("paged key weights: window must not be negative");
  if (batch->rows == 0 || cache->sequences == 0 || batch->max_rows == 0)
    return LFM3_OK;
  CHECK(CheckRows(q, q_stride, size_t(heads) * cache->dim,
                  "paged key weights: q or its stride"));
  if (!lse || !weights)
    return Invalid("paged key weights: lse and weights");
  if (!Aligned(4, {lse, weights}))
    return Invalid("paged key weights: lse or weights are not aligned");
  const PagedTables t = Tables(cache, batch);
  const size_t need = lfm3::paged_key_weights_workspace(t, cache->dim, heads);
  if (workspace_bytes < need || (need && !workspace) ||
      reinterpret_cast<uintptr_t>(workspace) % 256)
    return Invalid("paged key weights: workspace too small or not 256-byte "
                   "aligned");
  Memory memory;
  CHECK(memory.check(cache, false));
  CHECK(memory.check(batch));
  CHECK(memory.check(q, false,
                     "paged key weights: q is not on the current device"));
  if (need)
    CHECK(memory.check(workspace, false, "paged key weights: workspace is not "
                                         "on the current device"));
  CHECK(memory.check({lse, weights}, "paged key weights: lse or weights are "
                                     "not on the current device"));
  lfm3::PagedKeyWeightsArgs a{};
  a.t = t;
  a.q = q, a.lse = lse, a.weights = weights;
  a.ldq = q_stride;
  a.heads = heads;
  a.window = window;
  a.workspace = workspace;
  return Status(lfm3::launch_paged_key_weights(
      a, type, cache->dim, static_cast<cudaStream_t>(stream)));
}

int lfm3_cuda_paged_evict(const lfm3_paged_cache* cache,
                          const int32_t* out_table, int32_t* out_lengths,
                          float* weights, int32_t* kept, int keep, int recent,
                          void* stream) {
  CHECK(CheckCache(cache));
  if (!out_table || !out_lengths || !weights || !kept)
    return Invalid("paged evict: NULL array");
  if (!Aligned(4, {out_table, out_lengths, weights, kept}))
    return Invalid("paged evict: an array is not aligned");
  if (keep < 1 || recent < 0 || recent > keep)
    return Invalid("paged evict: keep must be positive, recent 0..keep");
  if (int64_t(cache->table_pages) * cache->page_rows < keep)
    return Invalid("paged evict: a sequence's pages hold fewer than keep rows");
  if (cache->sequences == 0)
    return LFM3_OK;
  Memory memory;
  CHECK(memory.check(cache));
  CHECK(memory.check(weights, false, "paged evict: weights are not on the "
                                     "current device"));
  CHECK(memory.check({out_table, out_lengths, kept},
                     "paged evict: an array is not on the current device"));
  lfm3::PagedEvictArgs a{};
  a.t = Tables(cache, nullptr);
  a.out_table = out_table;
  a.out_lengths = out_lengths;
  a.weights = weights;
  a.kept = kept;
  a.keep = keep;
  a.recent = recent;
  return Status(lfm3::launch_paged_evict(a, cache->dim,
                                         static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
