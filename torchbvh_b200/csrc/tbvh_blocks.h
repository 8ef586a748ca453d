// Block selection and block attention: geometry and plan shared by the
// selection kernels (tbvh_select.cu), the attention kernels
// (tbvh_attend_*.cu) and their C entries. No torch types.
//
// A block is a run of 64 consecutive leaves of a cloud's BVH order; block j is
// node j of the tree level six above the leaves, so its box is one row of
// node_aabbs. A tile is a run of 32 consecutive queries of a cloud in Morton
// order: spatial neighbours, whose selections mostly agree. The plan lists for
// every tile the union of its queries' blocks in ascending order, each with a
// 32-bit mask of the queries that selected it, and (for the backward pass) for
// every block the queries that selected it, in ascending tile order.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/torchbvh_b200.h"
#include "tbvh_common.cuh"

namespace tbvh {

constexpr int kBlockLevels = 6;
constexpr int kBlockLeaves = 1 << kBlockLevels;
constexpr int kTileQueries = 32;
constexpr int64_t kMostListTiles = (int64_t(1) << 32) / kTileQueries;  // of the backward lists, whose slots are 32 bits
constexpr int kMaxSelect = 32;
constexpr int kMaxBuckets = 64;

// One cloud: first packed point / node row / query / tile / block, and counts.
// Also the row of the host and device table of ragged calls (seven int64).
struct BlockCloud {
  int64_t p0, n, row0, q0, m, t0, b0;
};
static_assert(sizeof(BlockCloud) == 7 * 8, "table rows are seven int64");

__host__ __device__ inline int64_t blocks_of(int64_t n) { return (n + kBlockLeaves - 1) >> kBlockLevels; }
__host__ __device__ inline int64_t tiles_of(int64_t m) { return (m + kTileQueries - 1) / kTileQueries; }

struct BlockMap {
  const BlockCloud* table;  // device, ragged only
  int64_t n, m, rows;       // per cloud of a fixed-size batch
  int64_t num_tiles, num_blocks;
  int num_clouds;

  __device__ __forceinline__ BlockCloud uniform(int64_t b) const {
    return BlockCloud{b * n, n, b * rows, b * m, m, b * tiles_of(m), b * blocks_of(n)};
  }
  __device__ __forceinline__ BlockCloud of_cloud(int64_t b) const { return table == nullptr ? uniform(b) : table[b]; }
  __device__ __forceinline__ BlockCloud of_tile(int64_t t) const {
    if (table == nullptr) return uniform(num_clouds == 1 ? 0 : t / tiles_of(m));
    int lo = 0, hi = num_clouds - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (table[mid].t0 <= t) lo = mid; else hi = mid - 1;
    }
    return table[lo];
  }
  __device__ __forceinline__ BlockCloud of_block(int64_t j) const {
    if (table == nullptr) return uniform(num_clouds == 1 ? 0 : j / blocks_of(n));
    int lo = 0, hi = num_clouds - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (table[mid].b0 <= j) lo = mid; else hi = mid - 1;
    }
    return table[lo];
  }
};

// Plan arrays, carved from the caller's plan buffer.
struct BlockPlan {
  int* query_row;         // [tiles][32] packed query row, -1: none
  float* query_point;     // [tiles][3][32] its coordinates (0 past D and past the end)
  int* tile_count;        // [tiles] entries of each tile
  uint2* entries;         // [tiles][capacity] (block of the cloud, query mask)
  int64_t capacity;       // most entries a tile can have
  int64_t* query_begin;   // [blocks + 1] first list element of each block   (backward only from here)
  uint32_t* list;         // by block: query slots (32 * tile + lane), ascending
  int64_t* entry_begin;   // [blocks + 1] first entry of each block in `unsorted`  (scratch from here)
  int* entry_count;       // [blocks] entries, then fill cursors
  int* query_count;       // [blocks] queries
  uint2* unsorted;        // (tile, query mask) by block, in arrival order
};

// Host-side description of a selection, checked.
struct BlockSetup {
  BlockMap map;
  BlockPlan plan;
  int64_t total_points, total_queries, most_queries, most_blocks;  // most: of one cloud
};

// Checks the sizes and fills everything of `s` but the pointers.
int measure_blocks(const char* op, const tbvh_block_geometry* g, BlockSetup& s);
// Checks the struct and fills `s`; on failure sets tbvh_last_error() and returns the status.
int setup_blocks(const char* op, const tbvh_block_geometry* g, BlockSetup& s);
int blocks_fail(int code, const char* fmt, ...);
int blocks_cuda_fail(cudaError_t e, const char* op);

}  // namespace tbvh
