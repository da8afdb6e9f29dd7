// How the paged attention kernels share out a ragged batch, worked out on the
// device from starts and lengths (the host never reads them).
//
// The work is one line of equal units: per sequence, per row tile, per KV
// head, the key tiles that some row of the tile sees. Block b of a kernel
// takes units [b per, (b + 1) per) of that line, whatever sequences they fall
// in: every block does the same work for any mix of lengths. A stretch of one
// (sequence, row tile, KV head) inside a block's range is a segment. A segment
// that holds all the tiles writes the output; otherwise it leaves maxima, sums
// and unnormalised outputs in a slot of the workspace (a block has at most two
// such segments, its first and its last: slots 2 b and 2 b + 1). The block
// that holds a split stretch's first tiles (at most one such stretch begins in
// a block) also leaves a record of it, and the combine kernel merges record by
// record, in key order.
#pragma once
#include "paged.cuh"

namespace lfm3 {

// Single-token rows: keys in blocks of 16, one row tile per sequence.
constexpr int kDecodeKeys = 16;
constexpr int kDecodeCtas = 296;      // two per SM
constexpr int kDecodeMinUnits = 8;    // a block takes at least 128 keys
constexpr int kDecodeMaxGroup = 16;   // more heads per KV head: chunk kernel
// Chunks: tiles of 128 keys against pairs of 128-row tiles.
constexpr int kChunkKeys = 128;
constexpr int kChunkCtas = 148;       // one per SM
constexpr int kChunkRows = 128;       // (query, head of the group) rows, M

__host__ __device__ inline bool paged_single(int n, int group) {
  return n == 1 && group <= kDecodeMaxGroup;
}
// Queries of a row tile (its rows are query-major: query i / group).
__host__ __device__ inline int chunk_queries(int group) {
  return kChunkRows / group;
}

// First and last key that rows qlo .. qhi (of the sequence's new rows) see;
// last < first where they see none.
__host__ __device__ inline void paged_key_range(const PagedSequence& q,
                                                int window, int qlo, int qhi,
                                                int& first, int& last) {
  const int base = q.length - q.n;
  last = base + qhi;
  first = window > 0 && base + qlo >= window ? base + qlo - window + 1 : 0;
}

// Key units of a row tile (rows qlo .. qhi), from unit `lo`.
__host__ __device__ inline int paged_units(const PagedSequence& q, int window,
                                           int qlo, int qhi, int keys,
                                           int& lo) {
  int first, last;
  paged_key_range(q, window, qlo, qhi, first, last);
  lo = first / keys;
  return last < first ? 0 : last / keys - lo + 1;
}

// Single tokens share out their line in one of two ways. Equal shares cross
// from one stretch (a KV head of a sequence) to the next. A block pays for
// each segment (its queries, its first copies, the merge: 3.5 us, the time of
// kDecodeSegmentUnits units), so a stretch has that many empty places behind
// it in the line: a block of many short stretches gets fewer units (200
// sequences of 16 to 8000 keys, 4 KV heads: 233 us without, 131 us with).
// Rounding every stretch up to a multiple of the share instead gives a block
// one segment, at a larger share. That is taken when it is no slower: short or
// few sequences (8 rows of 100 keys 9.0 us padded, 10.9 us crossing, with the
// merge; of 1000 keys 11.5 and 13.0 us; where both are near, padded ones are up
// to 2 % slower), while 32 rows of 512 to 32768 keys would take 1.7
// times as long.
constexpr int kDecodeSegmentUnits = 10;
struct DecodePlan {
  int64_t share;
  int pad;    // every stretch's units are rounded up to a multiple of this
  int extra;  // empty places of the line behind each stretch
};

// Key units of a single-token sequence (0 for every other).
__device__ inline int decode_units(const PagedSequence& q, int group,
                                   int window) {
  int lo;
  return paged_single(q.n, group)
             ? paged_units(q, window, 0, 0, kDecodeKeys, lo)
             : 0;
}

// Pairs of row tiles of a chunk (0 for single tokens), and a pair's tiles.
__device__ inline int chunk_pairs(const PagedSequence& q, int group) {
  if (paged_single(q.n, group))
    return 0;
  const int queries = 2 * chunk_queries(group);
  return (q.n + queries - 1) / queries;
}
__device__ inline int chunk_units(const PagedSequence& q, int group,
                                  int window, int pair, int& lo) {
  const int queries = 2 * chunk_queries(group);
  return paged_units(q, window, pair * queries,
                     min(q.n, (pair + 1) * queries) - 1, kChunkKeys, lo);
}
// Places in the line of every step-th pair from pair `from` on (per KV head):
// its units, rounded up to a multiple of `pad`, and `extra` empty places, the
// time that a stretch takes beyond its tiles.
struct ChunkUnits {
  static constexpr bool kMany = true;
  int group, window, pad, extra;
  __device__ int rounded(int units) const {
    if (units == 0)
      return 0;
    return (pad == 1 ? units : (units + pad - 1) / pad * pad) + extra;
  }
  __device__ int64_t operator()(const PagedSequence& q, int from,
                                int step) const {
    const int pairs = chunk_pairs(q, group);
    int64_t sum = 0;
    int lo;
    for (int p = from; p < pairs; p += step)
      sum += rounded(chunk_units(q, group, window, p, lo));
    return sum;
  }
};

// Attention weights: pairs of 128-key tiles against blocks of columns, a
// column a (query, head of the group) of one KV head. The line runs over
// sequences, key pairs, KV heads and column blocks.
constexpr int kWeightKeys = 256;
constexpr int kWeightCtas = 148;  // one per SM

// Column blocks (chunk_queries queries each) of key pair `pair` in which some
// query sees some key, from block `lo`.
__device__ inline int weight_blocks(const PagedSequence& q, int group,
                                    int window, int pair, int& lo) {
  const int base = q.length - q.n, k0 = pair * kWeightKeys;
  const int k1 = min(k0 + kWeightKeys, q.length) - 1;
  const int first = max(0, k0 - base);
  int last = q.n - 1;
  if (window > 0 && int64_t(k1) + window - 1 - base < last)
    last = k1 + window - 1 - base;
  lo = first / chunk_queries(group);
  return last < first ? 0 : last / chunk_queries(group) - lo + 1;
}
__device__ inline int weight_pairs(const PagedSequence& q) {
  return q.n > 0 ? (q.length + kWeightKeys - 1) / kWeightKeys : 0;
}
struct WeightUnits {
  static constexpr bool kMany = true;
  int group, window;
  __device__ int64_t operator()(const PagedSequence& q, int from,
                                int step) const {
    const int pairs = weight_pairs(q), base = q.length - q.n;
    int64_t sum = 0;
    int lo, p = 0;
    if (window == 0) {
      // pairs that begin no later than the first new row: every block
      p = base < 0 ? 0 : min(pairs, base / kWeightKeys + 1);
      if (p > 0 && from == 0)
        sum = int64_t(p) * weight_blocks(q, group, window, 0, lo);
    } else if (base >= window) {
      p = (base - window + 1) / kWeightKeys;  // no row sees the pairs before
    }
    for (p += from; p < pairs; p += step)
      sum += weight_blocks(q, group, window, p, lo);
    return sum;
  }
};

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// (warp-wide)
__device__ inline DecodePlan decode_plan(const PagedTables& t, int group,
                                         int window) {
  int64_t units = 0;
  int stretches = 0;
  for (int s = threadIdx.x % 32; s < t.sequences; s += 32) {
    const int n = decode_units(paged_sequence(t, s), group, window);
    units += n;
    stretches += n > 0;
  }
  units = warp_sum64(units) * t.kv_heads;
  const int64_t pairs =
      int64_t(__reduce_add_sync(0xffffffffu, stretches)) * t.kv_heads;
  const int64_t crossing =
      max((units + kDecodeCtas - 1) / kDecodeCtas, int64_t(kDecodeMinUnits));
  if (pairs < kDecodeCtas) {
    const uint32_t left = uint32_t(kDecodeCtas - pairs);
    const int64_t padded =
        units >> 31 ? (units + left - 1) / left
                    : int64_t((uint32_t(units) + left - 1) / left);
    if (padded <= crossing + kDecodeSegmentUnits)
      return {max(padded, int64_t(kDecodeMinUnits)),
              int(max(padded, int64_t(kDecodeMinUnits))), 0};
  }
  return {max((units + pairs * kDecodeSegmentUnits + kDecodeCtas - 1) /
                  kDecodeCtas,
              int64_t(kDecodeMinUnits)),
          1, kDecodeSegmentUnits};
}

struct DecodeUnits {
  static constexpr bool kMany = false;
  int group, window, pad, extra;
  __device__ int rounded(int units) const {
    return units == 0 ? 0 : (units + pad - 1) / pad * pad + extra;
  }
  __device__ int64_t operator()(const PagedSequence& q, int, int) const {
    return rounded(decode_units(q, group, window));
  }
};

// Quotient of a unit number by a positive count (64-bit division is a long
// sequence of instructions, and lines of 2^32 units are rare).
__device__ __forceinline__ int64_t unit_div(int64_t a, int b) {
  return uint64_t(a) >> 32 ? a / b : int64_t(uint32_t(a) / uint32_t(b));
}

// The line of a batch (all members warp-wide); units(sequence, from, step) is
// every step-th part of a sequence's units from part `from` on. The first 32
// sequences' entries stay in registers, a lane each: for batches of up to 32
// the tables are read once. Searches go on where the last one ended (1500
// sequences of 16 to 100 keys: 1087 us from the front, 238 us). Where a
// sequence has many parts to sum (kMany), few sequences are summed by all lanes
// together, more a lane each.
constexpr int kFewSequences = 8;
template <typename Units>
struct PagedLine {
  const PagedTables& t;
  Units units;
  PagedSequence own;  // sequence `lane`
  int64_t own_units;
  int64_t total;  // units of the whole batch
  bool broken;    // this lane met a broken sequence
  int found = 0;  // the 32 sequences that find() ended at, and the units before
  int64_t found_sum = 0;

  __device__ PagedLine(const PagedTables& tables, Units u)
      : t(tables), units(u), own{0, 0, 0, false}, own_units(0), total(0),
        broken(false) {
    const int lane = threadIdx.x % 32;
    if (Units::kMany && t.sequences <= kFewSequences) {
      if (lane < t.sequences)
        own = paged_sequence(t, lane);
      broken = own.broken;
      reset(u);
      return;
    }
    for (int s = lane; s < t.sequences; s += 32) {
      const PagedSequence q = paged_sequence(t, s);
      const int64_t n = units(q, 0, 1);
      broken |= q.broken;
      total += n;
      if (s == lane) {
        own = q;
        own_units = n;
      }
    }
    total = warp_sum64(total);
  }

  // The same sequences (at most 32) with other units.
  __device__ void reset(Units u) {
    units = u;
    total = own_units = 0;
    // (sequences without rows have no units)
    for (unsigned left = __ballot_sync(0xffffffffu, own.n > 0); left;
         left &= left - 1) {
      const int s = __ffs(left) - 1;
      const PagedSequence q{0, __shfl_sync(0xffffffffu, own.n, s),
                            __shfl_sync(0xffffffffu, own.length, s), false};
      const int64_t n = warp_sum64(units(q, threadIdx.x % 32, 32));
      total += n;
      if (s == threadIdx.x % 32)
        own_units = n;
    }
  }

  // The sequence that holds unit `at` (never before the last one asked for),
  // its numbers, and the units before it. False past the end.
  __device__ bool find(int64_t at, int& s, PagedSequence& q,
                       int64_t& before) {
    const int lane = threadIdx.x % 32;
    int64_t sum = found_sum;
    for (int s0 = found; s0 < t.sequences; s0 += 32) {
      PagedSequence mine = own;
      int64_t u = own_units;
      if (s0 > 0) {
        mine = PagedSequence{0, 0, 0, false};
        u = 0;
        if (s0 + lane < t.sequences) {
          mine = paged_sequence(t, s0 + lane);
          u = units(mine, 0, 1);
        }
      }
      int64_t inc = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o)
          inc += x;
      }
      const unsigned past = __ballot_sync(0xffffffffu, sum + inc > at);
      if (past) {
        const int l = __ffs(past) - 1;
        s = s0 + l;
        q.row0 = __shfl_sync(0xffffffffu, mine.row0, l);
        q.n = __shfl_sync(0xffffffffu, mine.n, l);
        q.length = __shfl_sync(0xffffffffu, mine.length, l);
        q.broken = false;
        before = sum + __shfl_sync(0xffffffffu, inc - u, l);
        found = s0;
        found_sum = sum;
        return true;
      }
      sum += __shfl_sync(0xffffffffu, inc, 31);
    }
    return false;
  }
};

// Units per block for a line of `total` units over `ctas` blocks.
__device__ __forceinline__ int64_t paged_share(int64_t total, int ctas,
                                               int least) {
  return max((total + ctas - 1) / ctas, int64_t(least));
}

// One block's next piece of the chunks' line: units u0 .. u0 + count - 1 (of
// n_units, the first of them key tile `lo_unit`) of a pair of row tiles and a
// KV head, `units` of the line with its rounding, and the block's slot for it.
struct ChunkSegment {
  PagedSequence q;
  int seq, pair, h;
  int n_units, lo_unit, u0, count, units;
  int slot;
};
// The chunks' share and places (warp-wide), a similar choice. Equal shares
// cross stretches, each with `extra` empty places behind it (its queries, its
// first copies, its epilogue: about 8 us); prompts from position 0 are mostly
// short stretches (4 of 2000 rows: 279 us without the places, 144 us with).
// With more stretches than blocks, blocks may take whole ones instead, the same
// number each: that is no slower when they are about as long (chunks under a
// window of 256: 53 us crossing, 50.5 us whole), since nothing has to be
// merged. (24 chunks of 30 to 40 rows at 100 to 300 keys show the estimate's
// limits: 38 us whole, as it says, 35 us crossing.) With fewer, the smallest
// share with which rounded stretches still fit the blocks is taken, unless
// crossing shares save more than a second segment costs. That is worth 15 %
// where stretches are few and short (1024 f16 rows at depth 1000 48 us padded,
// 56 us crossing) and costs up to 5 % where they are long (512 FP32 rows at
// depth 8192, 32 stretches of 65 to 68 tiles, shares of 17 tiles instead of 15:
// 91 us padded, 88 us crossing) and 17 % for 200 f16 rows from position 0 (23
// and 19 us); over 72 batches of 1 to 4 chunks it costs 1 % on average.
__device__ inline int64_t chunk_plan(PagedLine<ChunkUnits>& line) {
  const PagedTables& t = line.t;
  const ChunkUnits& units = line.units;
  const int lane = threadIdx.x % 32, kvh = t.kv_heads, extra = units.extra;
  const int64_t crossing = paged_share(line.total * kvh, kChunkCtas, 1);
  if (t.sequences > 32 || crossing > 1 << 20)
    return crossing;
  int pairs = 0, some = 0;  // some: those that see a key
  if (lane < t.sequences) {
    pairs = chunk_pairs(line.own, units.group);
    const int idle = max(line.own.n - line.own.length, 0);
    if (line.own.length > 0)
      some = pairs - min(pairs, idle / (2 * chunk_queries(units.group)));
  }
  // (64 bits: the shares below hold every stretch, however many there are)
  const int64_t stretches = warp_sum64(int64_t(some) * kvh);
  if (stretches > kChunkCtas) {
    // whole stretches, `each` a block
    int top = 0, lo;
    for (unsigned left = __ballot_sync(0xffffffffu, some > 0); left;
         left &= left - 1) {
      const int s = __ffs(left) - 1;
      const PagedSequence q{0, __shfl_sync(0xffffffffu, line.own.n, s),
                            __shfl_sync(0xffffffffu, line.own.length, s),
                            false};
      const int n = __shfl_sync(0xffffffffu, pairs, s);
      for (int p = lane; p < n; p += 32)
        top = max(top, chunk_units(q, units.group, units.window, p, lo));
    }
    top = __reduce_max_sync(0xffffffffu, unsigned(top));
    const int64_t each = (stretches + kChunkCtas - 1) / kChunkCtas;
    if (each * (top + extra) > crossing + extra)
      return crossing;
    line.reset({units.group, units.window, top, 0});
    return each * top;
  }
  // lane l tries a share of least + l
  const int least =
      int((line.total * kvh - stretches * extra + kChunkCtas - 1) / kChunkCtas);
  const int share = max(least, 1) + lane;
  int blocks = 0, lo;
  for (unsigned left = __ballot_sync(0xffffffffu, some > 0); left;
       left &= left - 1) {
    const int s = __ffs(left) - 1;
    const PagedSequence q{0, __shfl_sync(0xffffffffu, line.own.n, s),
                          __shfl_sync(0xffffffffu, line.own.length, s), false};
    const int n = __shfl_sync(0xffffffffu, pairs, s);
    for (int p = 0; p < n; ++p)
      blocks += (chunk_units(q, units.group, units.window, p, lo) + share - 1) /
                share * kvh;
  }
  const unsigned fits = __ballot_sync(0xffffffffu, blocks <= kChunkCtas);
  if (fits == 0 || __ffs(fits) - 1 > extra)
    return crossing;
  const int pad = max(least, 1) + __ffs(fits) - 1;
  line.reset({units.group, units.window, pad, 0});
  return pad;
}

// The segment at unit `at` of a range that ends at `end` (warp-wide).
template <typename Line>
__device__ bool chunk_segment(Line& line, int64_t at, int64_t end,
                              ChunkSegment& g) {
  const int lane = threadIdx.x % 32, kvh = line.t.kv_heads;
  const ChunkUnits& u = line.units;
  const int group = u.group, window = u.window;
  int64_t before;
  if (at >= end || !line.find(unit_div(at, kvh), g.seq, g.q, before))
    return false;
  const int pairs = chunk_pairs(g.q, group);
  int64_t rel = at - before * kvh;
  for (int p0 = 0; p0 < pairs; p0 += 32) {
    int lo = 0;
    const int64_t mine =
        p0 + lane < pairs
            ? int64_t(u.rounded(chunk_units(g.q, group, window, p0 + lane,
                                            lo))) * kvh
            : 0;
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o)
        inc += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, inc > rel);
    if (past) {
      const int l = __ffs(past) - 1;
      rel -= __shfl_sync(0xffffffffu, inc - mine, l);
      g.pair = p0 + l;
      g.n_units = chunk_units(g.q, group, window, g.pair, g.lo_unit);
      const int stretch = u.rounded(g.n_units);
      g.h = int(unit_div(rel, stretch));
      g.u0 = int(rel - int64_t(g.h) * stretch);
      // (0 where the range begins in the empty places behind a stretch)
      g.count = int(max(min(int64_t(g.n_units - g.u0), end - at), int64_t(0)));
      g.units = g.u0 + g.count >= g.n_units ? stretch - g.u0 : g.count;
      return true;
    }
    rel -= __shfl_sync(0xffffffffu, inc, 31);
  }
  return false;
}

// The same for attention weights: inner units u0 .. u0 + count - 1 of n_units
// (KV head u / blocks, column block lo + u % blocks) of a pair of key tiles.
struct WeightSegment {
  PagedSequence q;
  int seq, pair;
  int blocks, lo;
  int n_units, u0, count;
  int slot;
};
template <typename Line>
__device__ bool weight_segment(Line& line, int group, int window,
                               int64_t at, int64_t end, WeightSegment& g) {
  const int lane = threadIdx.x % 32, kvh = line.t.kv_heads;
  int64_t before;
  if (at >= end || !line.find(unit_div(at, kvh), g.seq, g.q, before))
    return false;
  const int pairs = weight_pairs(g.q);
  int64_t rel = at - before * kvh;
  for (int p0 = 0; p0 < pairs; p0 += 32) {
    int lo = 0;
    const int64_t mine =
        p0 + lane < pairs
            ? int64_t(weight_blocks(g.q, group, window, p0 + lane, lo)) * kvh
            : 0;
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o)
        inc += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, inc > rel);
    if (past) {
      const int l = __ffs(past) - 1;
      rel -= __shfl_sync(0xffffffffu, inc - mine, l);
      g.pair = p0 + l;
      g.blocks = weight_blocks(g.q, group, window, g.pair, g.lo);
      g.n_units = g.blocks * kvh;
      g.u0 = int(rel);
      g.count = int(min(int64_t(g.n_units - g.u0), end - at));
      return true;
    }
    rel -= __shfl_sync(0xffffffffu, inc, 31);
  }
  return false;
}

// A stretch that several blocks share: `parts` slots, the first `slot`, then
// every second one from the next even number on (the blocks after the first
// begin with it). parts 0: none begins in the block.
struct PagedRecord {
  int parts, slot;
  int row0;  // tensor row of the sequence's first new row
  int n;     // its new rows
  int pair, h;
};
__device__ __forceinline__ int record_slot(const PagedRecord& r, int part) {
  return part == 0 ? r.slot : (r.slot & ~1) + 2 * part;
}
// The record of a segment at unit `at` (units of its stretch: n_units) that
// starts the stretch but does not end it.
__device__ __forceinline__ PagedRecord paged_record(int64_t at, int64_t share,
                                                    int slot, int n_units,
                                                    const PagedSequence& q,
                                                    int pair, int h) {
  const int64_t past = at + n_units - 1 - int64_t(blockIdx.x) * share;
  return {int(past / share) + 1, slot, q.row0, q.n, pair, h};
}

// ---- numbers of the softmax ----------------------------------------------
// Scores are kept in base 2: x = (q k) rsqrt(dim) log2 e.
constexpr float kLog2e = 1.44269504088896341F;
constexpr float kLn2 = 0.693147180559945309F;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The power of two that brings a row's largest magnitude into [2^14, 2^15),
// so that its fp16 terms neither overflow nor lose bits (1 for rows of zeros
// or with values that are not finite).
__device__ __forceinline__ float row_scale(float top) {
  const int e = int(__float_as_uint(top) >> 23);
  if (!(top > 0) || e == 255)
    return 1.0F;
  return __uint_as_float(uint32_t(min(127 + 14 - (e - 127), 254)) << 23);
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 bits_half2(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

}  // namespace lfm3
