// TMA tensor maps: Q8_0 weight rows viewed as [rows][row_bytes / 8] 8-byte
// elements (one copy lands a box of rows as dense shared-memory rows of the
// box width; rows and columns past the matrix read as zeros), and fp16
// activation rows with the 64-byte swizzle of the tcgen05 operand layout.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace lfm3 {

// Encodes a map over Q8_0 rows viewed as [rows][row_bytes / 8] 8-byte
// elements (row_bytes a multiple of 16), boxes of box_bytes (a multiple of
// 16, <= 2048) x box_rows: one copy lands box_rows dense rows of box_bytes.
cudaError_t encode_q8_rows(CUtensorMap* map, const void* base, size_t row_bytes,
                           int rows, int box_bytes, int box_rows);

// Encodes a map over fp16 activations [rows][cols] (row pitch cols * 2
// bytes) with boxes of box_rows x box_cols (box_cols * 2 == 64) and the
// 64-byte swizzle the tcgen05 K-major operand layout expects.
cudaError_t encode_activation_map(CUtensorMap* map, const void* base, int rows,
                                  int cols, int box_rows, int box_cols);

// Encodes a map over a pool of fp16 rows [rows][heads * dim] (dim a multiple
// of 64) as [heads * dim / 64][rows][64] with boxes of box_slabs x box_rows x
// 64 and the 128-byte swizzle: one copy lands box_rows of a head as dim / 64
// (box_slabs) slabs of 128-byte rows. Box coordinates: 0, row, slab.
cudaError_t encode_pool_map(CUtensorMap* map, const void* base, int rows,
                            int heads, int dim, int box_rows, int box_slabs);

// Encodes a map over fp16 rows [rows][kv_heads][group][dim] as [kv_heads]
// [dim / 64][rows][group][64] with boxes of box_rows rows of one KV head and
// slab, 128-byte swizzle: one copy lands a KV head's (row, head) pairs as
// 128-byte rows. Box coordinates: 0, 0, row, slab, KV head.
cudaError_t encode_group_map(CUtensorMap* map, const void* base, int rows,
                             int kv_heads, int group, int dim, int box_rows);

// The weight and activation maps from a process-wide cache keyed by every
// encode argument (a hit is exactly the map the encoder would write).
cudaError_t cached_q8_rows(CUtensorMap* map, const void* base, size_t row_bytes,
                           int rows, int box_bytes, int box_rows);
cudaError_t cached_activation_map(CUtensorMap* map, const void* base, int rows,
                                  int cols, int box_rows, int box_cols);

}  // namespace lfm3
