// Paged key/value cache held in 4 bits (cache.cu): its layout, and what its kernels take.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "cache_runs.cuh"
#include "lsx.h"

namespace lsx {

constexpr int kCacheGroup = 64;     // elements that share a step and a zero
constexpr int kMaxCacheDim = 256;   // widest head
constexpr int kMaxListed = 1024;    // sequences that one call forks or extends
constexpr int kMaxFreed = 65536;    // and empties: each is looked for among those before it

// The bytes of a cell for heads of `dim` elements, and where its parts start.
__host__ __device__ constexpr int cell_bytes(int dim) { return 18 * dim; }
__host__ __device__ constexpr int cell_values(int dim) { return 8 * dim; }
__host__ __device__ constexpr int cell_key_steps(int dim) { return 16 * dim; }
__host__ __device__ constexpr int cell_value_steps(int dim) { return 17 * dim; }

// The byte that holds key elements d and d + 1 (d even; d in the low bits) of position t.
__host__ __device__ inline int key_byte(int t, int d) {
    return (d / 64 * 32 + t % 8 * 4 + d % 64 / 16) * 16 + t / 8 * 8 + d % 16 / 2;
}
// The byte that holds value elements d and d + 8 (d % 16 < 8; d in the low bits) of position t.
__host__ __device__ inline int value_byte(int dim, int t, int d) {
    return cell_values(dim) + (d / 64 * 32 + d % 8 * 4 + t % 8 / 2) * 16 + d / 16 % 4 * 4 + t % 2 * 2 + t / 8;
}
// The step of group g of position t within the keys' or values' steps; its zero lies 4 bytes on.
__host__ __device__ inline int step_byte(int t, int g) { return g * 64 + t % 8 / 2 * 16 + t / 8 * 8 + t % 2 * 2; }

// One layer's pages and the sequences in them (lsx_cache_view).
struct CacheView {
    uint8_t* pages;
    const int32_t* tables;
    const int32_t* lengths;
    uint32_t page_count, page_size, kv_heads, dim, table_rows, table_width;
};

// The rows of a call: sequence b of `count` (row sequences[b] of the tables, b without
// the list) has rows starts[b] .. starts[b + 1] (row b alone without them), which are its
// last positions.
struct CacheRows {
    const int32_t* sequences;
    const int32_t* starts;
    uint32_t count, rows;
};

}  // namespace lsx
