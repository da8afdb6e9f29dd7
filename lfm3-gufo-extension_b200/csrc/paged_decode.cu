// Attention of single new tokens over paged keys and values: the sequences of
// a batch with one new row (and at most 16 heads to a KV head).
//
// HBM bound: each visible key and value is read once for the G query heads of
// its KV head, 2 G flops a byte. So the kernel keeps bytes in flight and the
// arithmetic out of the way. Blocks of 128 threads, two to an SM, take equal
// shares of the batch's 16-key blocks (paged_plan.cuh). Inside a block the
// warps are independent: warp w takes blocks w, w + 4, ... of the segment
// through its own ring of buffers, filled by TMA (one copy lands a head's 16
// rows of K or V; 16 divides page_rows, so a block lies in one page), and
// keeps its own online softmax; the four states merge at the segment's end.
// Both products run on mma.sync m16n8k16 with FP32 accumulation: S^T = K Q^T
// with 16 keys as M and the heads (padded to 8 or 16) as N, O^T += V^T P^T
// with the dimensions as M, the probability fragments transposed in registers.
// (tcgen05 would need 128 keys a step and its accumulator read back through
// tensor memory for 8 columns of work; the tensor pipe is idle here anyway.)
// FP32 queries enter as two fp16 terms and their probabilities too (22 bits);
// 16-bit queries are exact in one term and the probabilities round to fp16
// once, which is below their output's own rounding.
// Measured with the merge: 32 rows over 512 to 32768 keys (597 MB) 103 us,
// 5.8 TB/s (FP32 rows 105 us); 8 rows over 85 to 1995 keys 15 us, all of it
// latency (launches, tables, first copies, merge).
#include "kernels.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "tensor_map.hpp"

namespace lfm3 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
// The largest probability so far is 2^7: small ones stay clear of fp16's
// subnormals.
constexpr float kTopExponent = 7.0F;

template <int DIM, int NT, int TERMS>
struct __align__(1024) DecodeSmem {
  // bytes in flight: 96 KB of K and V a block, 192 KB an SM
  static constexpr int kStages = 3 * 128 / DIM;
  static constexpr int kTile = 16 * DIM * 2;  // K or V bytes of a block
  uint8_t ring[kWarps][kStages][2][kTile];
  __half q[TERMS][8 * NT * DIM];
  float c[8 * NT];  // score factor of each head
  float wm[kWarps][8 * NT], wl[kWarps][8 * NT], ws[kWarps][8 * NT];
  float m[8 * NT], l[8 * NT];
  uint64_t full[kWarps][kStages];
  static_assert(kWarps * 8 * NT * DIM * 4 <= sizeof(ring),
                "the merge's outputs fit the ring");
};

// 16-byte piece `piece` of row `row`: of a query row (DIM wide), and of a TMA
// tile (slabs of [16][64] with the 128-byte swizzle).
template <int DIM>
__device__ __forceinline__ int at_q(int row, int piece) {
  return row * DIM + ((piece ^ (row & 7)) << 3);
}
__device__ __forceinline__ int at_tile(int row, int piece) {
  return (piece >> 3) * 2048 + row * 128 + (((piece ^ row) & 7) << 4);
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;"
               : "=r"(d)
               : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_half2(__half lo, __half hi) {
  return uint32_t(__half_as_ushort(lo)) |
         (uint32_t(__half_as_ushort(hi)) << 16);
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p)));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile(
      "ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(smem_addr(p)));
}
__device__ __forceinline__ void ldsm_x2(uint32_t (&r)[2], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
               : "=r"(r[0]), "=r"(r[1])
               : "r"(smem_addr(p)));
}

template <typename T, int DIM, int NT>
__global__ void __launch_bounds__(kThreads, 2)
    paged_decode_kernel(const __grid_constant__ PagedAttentionArgs a) {
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  using Smem = DecodeSmem<DIM, NT, TERMS>;
  constexpr int kStages = Smem::kStages;
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int kvh = a.t.kv_heads, group = a.heads / kvh;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i)
      mbar_init(&s.full[warp][i], 1);
    fence_barrier_init();
    prefetch_map(&a.kmap16);
    prefetch_map(&a.vmap16);
  }
  // what earlier kernels wrote is there; kernels launched behind this one may
  // start once every block is past this point
  grid_dependency_wait();
  allow_dependents();
  const DecodePlan plan = decode_plan(a.t, group, a.window);
  const DecodeUnits units{group, a.window, plan.pad, plan.extra};
  PagedLine line(a.t, units);
  if (line.broken && blockIdx.x == 0 && warp == 0)
    report_error(kErrPagedTable);
  const int64_t total = line.total * kvh;
  const int64_t share = plan.share;
  const int64_t begin = share * blockIdx.x, end = min(begin + share, total);
  PagedRecord record{0, 0, 0, 0, 0, 0};
  uint32_t used = 0;  // buffers this warp has filled so far
  const int fg = lane / 4, cq = lane % 4, mj = lane / 8, mrow = lane % 8;
  __syncwarp();

  for (int64_t at = begin, next; at < end; at = next) {
    // ---- the segment: units [u0, u0 + count) of KV head h of sequence seq
    int seq, lo_unit;
    PagedSequence q{};
    int64_t before;
    if (!line.find(unit_div(at, kvh), seq, q, before))
      break;
    const int n_units = paged_units(q, a.window, 0, 0, kDecodeKeys, lo_unit);
    const int64_t rel = at - before * kvh;
    const int stretch = units.rounded(n_units);
    const int h = int(unit_div(rel, stretch));
    const int u0 = int(rel - int64_t(h) * stretch);
    if (u0 >= n_units) {  // the empty places behind a stretch
      next = at + stretch - u0;
      continue;
    }
    const int count = int(min(int64_t(n_units - u0), end - at));
    next = at + (u0 + count == n_units ? stretch - u0 : count);
    // ---- the group's queries are on their way while the page ids come
    const int r = q.row0;
    constexpr int kPerWarp = 8 * NT / kWarps;
    float xq[kPerWarp][DIM / 32];
#pragma unroll
    for (int jj = 0; jj < kPerWarp; ++jj) {
      const int j = warp + jj * kWarps;
#pragma unroll
      for (int i = 0; i < DIM / 32; ++i)
        xq[jj][i] =
            j < group
                ? to_float(static_cast<const T*>(
                      a.q)[size_t(r) * a.ldq + size_t(h * group + j) * DIM +
                           lane + 32 * i])
                : 0.0F;
    }
    int first_key, last_key;
    paged_key_range(q, a.window, 0, 0, first_key, last_key);
    const int mine = (count - warp + kWarps - 1) / kWarps;  // this warp's
    // page ids are read one lane per block, 32 blocks ahead of their use
    const auto pool_row = [&](int i) {  // block i of this warp
      const int key = (lo_unit + u0 + warp + i * kWarps) * kDecodeKeys;
      int row = paged_row(a.t, a.t.table, seq, key);
      if (row < 0) {
        report_error(kErrPagedTable);
        row = 0;
      }
      return row;
    };
    int rows = lane < mine ? pool_row(lane) : 0;
    const auto issue = [&](int i) {  // warp-wide
      if (i >= mine)
        return;
      if (i % 32 == 0 && i > 0)
        rows = i + lane < mine ? pool_row(i + lane) : 0;
      const int row = __shfl_sync(0xffffffffu, rows, i % 32);
      if (lane == 0) {
        const int st = (used + i) % kStages;
        mbar_arrive_expect_tx(&s.full[warp][st], 2 * Smem::kTile);
        tma_load_3d(s.ring[warp][st][0], &a.kmap16, 0, row, h * (DIM / 64),
                    &s.full[warp][st]);
        tma_load_3d(s.ring[warp][st][1], &a.vmap16, 0, row, h * (DIM / 64),
                    &s.full[warp][st]);
      }
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i)
      issue(i);

    // ---- the queries, each scaled to fp16's range by a power of two
#pragma unroll
    for (int jj = 0; jj < kPerWarp; ++jj) {
      const int j = warp + jj * kWarps;
      const float(&x)[DIM / 32] = xq[jj];
      float top = 0;
#pragma unroll
      for (int i = 0; i < DIM / 32; ++i)
        top = fmaxf(top, fabsf(x[i]));
      const float scale = row_scale(warp_max(top));
#pragma unroll
      for (int i = 0; i < DIM / 32; ++i) {
        const int d = lane + 32 * i;
        const SplitPair t = split_value(x[i] * scale);
        s.q[0][at_q<DIM>(j, d / 8) + d % 8] = t.hi;
        if constexpr (TERMS == 2)
          s.q[TERMS - 1][at_q<DIM>(j, d / 8) + d % 8] = t.lo;
      }
      if (lane == 0)
        s.c[j] = rsqrtf(float(DIM)) * kLog2e / scale;
    }
    __syncthreads();
    uint32_t qb[TERMS][NT][DIM / 16][2];
    float c[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int ks = 0; ks < DIM / 16; ++ks)
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
          ldsm_x2(qb[t][nt][ks],
                  &s.q[t][at_q<DIM>(8 * nt + mrow, 2 * ks + (mj & 1))]);
      c[nt][0] = s.c[8 * nt + 2 * cq];
      c[nt][1] = s.c[8 * nt + 2 * cq + 1];
    }
    float mrun[NT][2], lrun[NT][2], o[NT][DIM / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mrun[nt][0] = mrun[nt][1] = -INFINITY;
      lrun[nt][0] = lrun[nt][1] = 0;
#pragma unroll
      for (int mt = 0; mt < DIM / 16; ++mt)
        o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0;
    }

    bool ok = true;
    for (int i = 0; i < mine && ok; ++i) {
      const int st = (used + i) % kStages;
      ok = __all_sync(0xffffffffu,
                      mbar_wait(&s.full[warp][st], ((used + i) / kStages) & 1,
                                kErrPagedWait));
      if (!ok)
        break;
      const uint8_t* tk = s.ring[warp][st][0];
      uint8_t* tv = s.ring[warp][st][1];
      // visible keys of the block: lo <= key < hi
      const int key0 = (lo_unit + u0 + warp + i * kWarps) * kDecodeKeys;
      const int lo = first_key - key0, hi = last_key + 1 - key0;
      if (lo > 0 || hi < 16) {
        // other rows of the page may hold anything: their values become 0 (a
        // probability of 0 times a NaN would still be NaN)
        for (int p = lane; p < 16 * DIM / 8; p += 32) {
          const int row = p / (DIM / 8);
          if (row < lo || row >= hi)
            *reinterpret_cast<uint4*>(tv + at_tile(row, p % (DIM / 8))) =
                make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();  // ordered before the TMA that refills the buffer
        __syncwarp();
      }
      // ---- S^T = K Q^T, two accumulation chains
      float acc[NT][2][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          acc[nt][0][x] = acc[nt][1][x] = 0;
#pragma unroll
      for (int ks = 0; ks < DIM / 16; ++ks) {
        uint32_t f[4];
        ldsm_x4(f, tk + at_tile((mj & 1) * 8 + mrow, 2 * ks + (mj >> 1)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int t = 0; t < TERMS; ++t)
            mma_f16(acc[nt][TERMS == 2 ? t : ks & 1], f, qb[t][nt][ks][0],
                    qb[t][nt][ks][1]);
      }
      // this thread: keys fg and fg + 8, heads 8 nt + 2 cq and + 1
      uint32_t ph[NT][2], pl[NT][2];
      float alpha[NT][2];
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = acc[nt][0][e] + acc[nt][1][e];
        if (fg < lo || fg >= hi)
          x[0] = x[1] = -INFINITY;
        if (fg + 8 < lo || fg + 8 >= hi)
          x[2] = x[3] = -INFINITY;
        float pr[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // Rounded to FP32 before the maximum is taken from them: past 2^24
          // one fused operation would leave the maximum's rounding in the
          // exponent.
          x[e] = __fmul_rn(x[e], c[nt][e]);
          x[e + 2] = __fmul_rn(x[e + 2], c[nt][e]);
          float top = fmaxf(x[e], x[e + 2]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          top = fmaxf(mrun[nt][e], top - kTopExponent);
          // (keys whose scores are all -infinity weigh nothing)
          const float ref = top == -INFINITY ? 0.0F : top;
          alpha[nt][e] = ex2(mrun[nt][e] - ref);
          moved |= top > mrun[nt][e];
          mrun[nt][e] = top;
          pr[e] = ex2(x[e] - ref);
          pr[e + 2] = ex2(x[e + 2] - ref);
          lrun[nt][e] = lrun[nt][e] * alpha[nt][e] + (pr[e] + pr[e + 2]);
        }
        const SplitPair p0 = split_value(pr[0]), p1 = split_value(pr[1]);
        const SplitPair p2 = split_value(pr[2]), p3 = split_value(pr[3]);
        ph[nt][0] = transpose8x8(pack_half2(p0.hi, p1.hi));
        ph[nt][1] = transpose8x8(pack_half2(p2.hi, p3.hi));
        if constexpr (TERMS == 2) {
          pl[nt][0] = transpose8x8(pack_half2(p0.lo, p1.lo));
          pl[nt][1] = transpose8x8(pack_half2(p2.lo, p3.lo));
        }
      }
      if (__any_sync(0xffffffffu, moved))
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < DIM / 16; ++mt) {
            o[nt][mt][0] *= alpha[nt][0];
            o[nt][mt][1] *= alpha[nt][1];
            o[nt][mt][2] *= alpha[nt][0];
            o[nt][mt][3] *= alpha[nt][1];
          }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int mt = 0; mt < DIM / 16; ++mt) {
        uint32_t f[4];
        ldsm_x4_trans(f, tv + at_tile((mj >> 1) * 8 + mrow, 2 * mt + (mj & 1)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(o[nt][mt], f, ph[nt][0], ph[nt][1]);
          if constexpr (TERMS == 2)
            mma_f16(o[nt][mt], f, pl[nt][0], pl[nt][1]);
        }
      }
      __syncwarp();  // the buffer is free
      issue(i + kStages);
    }
    if (__syncthreads_or(!ok)) {
      // a copy never landed: the block gives up once those it issued have
      // (again within the waits' limit)
      for (int i = 0; i < kStages && i < mine; ++i)
        mbar_wait(&s.full[warp][(used + i) % kStages],
                  ((used + i) / kStages) & 1, kErrPagedWait);
      record.parts = 0;
      break;
    }
    used += mine > 0 ? mine : 0;

    // ---- the warps' states merged (the ring's buffers hold their outputs)
    float* wo = reinterpret_cast<float*>(s.ring);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // (each lane's sum holds its own keys)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
          lrun[nt][e] += __shfl_xor_sync(0xffffffffu, lrun[nt][e], off);
        float* w = wo + (warp * 8 * NT + 8 * nt + 2 * cq + e) * DIM;
#pragma unroll
        for (int mt = 0; mt < DIM / 16; ++mt) {
          w[mt * 16 + fg] = o[nt][mt][e];
          w[mt * 16 + fg + 8] = o[nt][mt][e + 2];
        }
        if (fg == 0) {
          s.wm[warp][8 * nt + 2 * cq + e] = mrun[nt][e];
          s.wl[warp][8 * nt + 2 * cq + e] = lrun[nt][e];
        }
      }
    }
    __syncthreads();
    if (tid < group) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        top = fmaxf(top, s.wm[w][tid]);
      float l = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        // a warp without keys, or with none but scores of -inf, has maximum
        // -inf and weight 0
        const float f = s.wm[w][tid] == -INFINITY ? 0.0F
                                                  : ex2(s.wm[w][tid] - top);
        s.ws[w][tid] = f;
        l = fmaf(s.wl[w][tid], f, l);
      }
      s.m[tid] = top;
      s.l[tid] = l;
    }
    __syncthreads();
    const bool whole = count == n_units;
    const int slot = 2 * blockIdx.x + (at > begin ? 1 : 0);
    if (!whole && u0 == 0)
      record = paged_record(at, share, slot, n_units, q, 0, h);
    float* po = a.decode_part + size_t(slot) * group * DIM;
    float* pm = a.decode_part + size_t(2 * kDecodeCtas) * group * DIM +
                size_t(slot) * group * 2;
    for (int i = tid; i < group * DIM; i += kThreads) {
      const int j = i / DIM, d = i % DIM, head = h * group + j;
      float y = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        y = fmaf(wo[(w * 8 * NT + j) * DIM + d], s.ws[w][j], y);
      if (!whole) {
        po[i] = y;
        if (d < 2)
          pm[j * 2 + d] = d ? s.l[j] : s.m[j];
        continue;
      }
      y = s.l[j] == 0 ? 0.0F : y / s.l[j];  // 0: no key but scores of -inf
      if (a.gate)
        y /= 1 + expf(-to_float(
                 static_cast<const T*>(a.gate)[size_t(r) * a.ldg + head]));
      static_cast<T*>(a.out)[size_t(r) * a.ldo + size_t(head) * DIM + d] =
          from_float<T>(y);
      if (a.lse && d == 0)
        a.lse[size_t(r) * a.heads + head] = (s.m[j] + log2f(s.l[j])) * kLn2;
    }
    // the next segment's copies come after these reads and writes
    fence_proxy_async();
    __syncthreads();
  }
  // rows that see no key (idle sequences)
  for (int j = blockIdx.x; j < a.t.sequences; j += gridDim.x) {
    const PagedSequence q = paged_sequence(a.t, j);
    if (paged_single(q.n, group) && decode_units(q, group, a.window) == 0) {
      for (int i = tid; i < a.heads * DIM; i += kThreads)
        static_cast<T*>(a.out)[size_t(q.row0) * a.ldo + i] = from_float<T>(0);
      for (int i = tid; a.lse && i < a.heads; i += kThreads)
        a.lse[size_t(q.row0) * a.heads + i] = -INFINITY;
    }
  }
  if (tid == 0)
    reinterpret_cast<PagedRecord*>(
        a.decode_part +
        size_t(2 * kDecodeCtas) * group * (DIM + 2))[blockIdx.x] = record;
}

template <typename T, int DIM, int NT>
cudaError_t launch(const PagedAttentionArgs& a, cudaStream_t stream) {
  const auto kernel = paged_decode_kernel<T, DIM, NT>;
  const int smem =
      int(sizeof(DecodeSmem<DIM, NT, sizeof(T) == 4 ? 2 : 1>)) + 1024;
  if (cudaError_t e =
          ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem))
    return e;
  return launch_kernel(kernel, dim3(kDecodeCtas), dim3(kThreads), smem, stream,
                       true, a);
}
template <typename T>
cudaError_t launch(const PagedAttentionArgs& a, int dim, cudaStream_t stream) {
  const bool wide = a.heads / a.t.kv_heads > 8;
  if (dim == 64)
    return wide ? launch<T, 64, 2>(a, stream) : launch<T, 64, 1>(a, stream);
  return wide ? launch<T, 128, 2>(a, stream) : launch<T, 128, 1>(a, stream);
}

}  // namespace

size_t paged_decode_floats(int dim, int group) {
  return group > kDecodeMaxGroup ? 0
                                 : size_t(2 * kDecodeCtas) * group * (dim + 2) +
                                       kDecodeCtas * sizeof(PagedRecord) / 4;
}

cudaError_t launch_paged_decode(const PagedAttentionArgs& a, uint32_t type,
                                int dim, cudaStream_t stream) {
  return type == LFM3_F32   ? launch<float>(a, dim, stream)
         : type == LFM3_F16 ? launch<__half>(a, dim, stream)
                            : launch<__nv_bfloat16>(a, dim, stream);
}

}  // namespace lfm3
