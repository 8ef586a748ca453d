// Block selection: for every query the blocks of 64 leaves whose boxes are
// nearest, and the plan that block attention reads (tbvh_blocks.h).
//
// score(q, j) = sum_a max(lo_ja - q_a, max(q_a - hi_ja, 0))^2, each operation
// rounded in float32 (no contraction), so that any implementation that rounds
// the same way selects the same blocks. All steps are monotone: a box inside
// another never scores lower, in float32 too, which is what makes pruning by
// the inner nodes exact. Ties go to the lower block: keys are (score bits,
// block) pairs, and a node's key holds its first block, so a node whose score
// ties the k-th best is entered only if it could still win by index. Coincident
// clouds, where every block scores the same, therefore end after k blocks.
//
// This file is compiled without fast math: scores keep subnormals.
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "tbvh_blocks.h"
#include "tbvh_kernels.h"

namespace tbvh {

int blocks_fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return record_error(code, buf);
}

int blocks_cuda_fail(cudaError_t e, const char* op) {
  return blocks_fail(TBVH_ERR_CUDA, "%s: CUDA error %s (%s)", op, cudaGetErrorName(e), cudaGetErrorString(e));
}

namespace {

size_t pad256(size_t v) { return (v + 255) / 256 * 256; }

struct PlanSizes {
  size_t rows, points, count, entries, begin, counts, list, unsorted;
};

PlanSizes plan_sizes(int64_t tiles, int64_t capacity, int64_t blocks, int64_t picks, bool backward) {
  PlanSizes p{};
  p.rows = pad256(size_t(tiles) * kTileQueries * sizeof(int));
  p.points = pad256(size_t(tiles) * 3 * kTileQueries * sizeof(float));
  p.count = pad256(size_t(tiles) * sizeof(int));
  p.entries = pad256(size_t(tiles) * size_t(capacity) * sizeof(uint2));
  if (backward) {
    p.begin = pad256(size_t(blocks + 1) * sizeof(int64_t));
    p.counts = pad256(size_t(blocks) * sizeof(int));
    p.list = pad256(size_t(picks) * sizeof(uint32_t));
    p.unsorted = p.entries;
  }
  return p;
}

size_t plan_total(const PlanSizes& p) {
  return p.rows + p.points + p.count + p.entries + 2 * p.begin + 2 * p.counts + p.list + p.unsorted;
}

PlanSizes plan_sizes(const BlockSetup& s, const tbvh_block_geometry* g) {
  return plan_sizes(s.map.num_tiles, s.plan.capacity, s.map.num_blocks, s.total_queries * g->num_blocks,
                    g->backward != 0);
}

}  // namespace

// Sizes only: everything but the pointers.
int measure_blocks(const char* op, const tbvh_block_geometry* g, BlockSetup& s) {
  s = BlockSetup{};
  if (g == nullptr) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: geometry is NULL", op);
  if (g->dim != 2 && g->dim != 3) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: D must be 2 or 3", op);
  if (g->num_blocks < 1 || g->num_blocks > kMaxSelect)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: num_blocks must be 1 to %d", op, kMaxSelect);
  if (g->num_clouds < 1 || g->num_clouds > INT_MAX)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: number of clouds must be in [1, 2^31)", op);
  int64_t most_blocks = 0, most_queries = 0;
  BlockMap& map = s.map;
  map.num_clouds = int(g->num_clouds);
  if (g->points_per_cloud > 0) {
    if (g->points_per_cloud > INT_MAX || g->num_clouds * g->points_per_cloud > INT_MAX)
      return blocks_fail(TBVH_ERR_BAD_ARG, "%s: total point count must fit in signed int32", op);
    if (g->queries_per_cloud < 0 || g->queries_per_cloud > INT_MAX ||
        g->num_clouds * g->queries_per_cloud > INT_MAX)
      return blocks_fail(TBVH_ERR_BAD_ARG, "%s: total query count must fit in signed int32", op);
    map.n = g->points_per_cloud;
    map.m = g->queries_per_cloud;
    map.rows = real_node_count(map.n);
    map.num_tiles = g->num_clouds * tiles_of(map.m);
    map.num_blocks = g->num_clouds * blocks_of(map.n);
    most_blocks = blocks_of(map.n);
    most_queries = map.m;
    s.total_points = g->num_clouds * map.n;
    s.total_queries = g->num_clouds * map.m;
  } else {
    const auto* t = reinterpret_cast<const BlockCloud*>(g->table_host);
    if (t == nullptr) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: ragged clouds need a host table", op);
    BlockCloud want{};
    for (int64_t b = 0; b < g->num_clouds; ++b) {
      const BlockCloud& c = t[b];
      if (c.n < 1 || c.m < 0 || c.n > INT_MAX || c.m > INT_MAX || c.p0 != want.p0 || c.row0 != want.row0 ||
          c.q0 != want.q0 || c.t0 != want.t0 || c.b0 != want.b0)
        return blocks_fail(TBVH_ERR_BAD_ARG, "%s: the host table is not one of tbvh_block_table", op);
      want.p0 += c.n;
      want.row0 += real_node_count(c.n);
      want.q0 += c.m;
      want.t0 += tiles_of(c.m);
      want.b0 += blocks_of(c.n);
      if (want.p0 > INT_MAX) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: total point count must fit in signed int32", op);
      if (want.q0 > INT_MAX) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: total query count must fit in signed int32", op);
      if (blocks_of(c.n) > most_blocks) most_blocks = blocks_of(c.n);
      if (c.m > most_queries) most_queries = c.m;
    }
    map.num_tiles = want.t0;
    map.num_blocks = want.b0;
    s.total_points = want.p0;
    s.total_queries = want.q0;
  }
  // Small clouds have a tile each: more tiles than 32-bit query slots reach are fewer than 2^31 queries.
  if (g->backward && map.num_tiles > kMostListTiles)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: too many clouds for the backward lists (at most 2^27 tiles of %d queries)",
                       op, kTileQueries);
  s.most_queries = most_queries;
  s.most_blocks = most_blocks;
  s.plan.capacity = (most_queries < kTileQueries ? most_queries : kTileQueries) * g->num_blocks;
  if (s.plan.capacity > most_blocks) s.plan.capacity = most_blocks;
  return TBVH_OK;
}

int setup_blocks(const char* op, const tbvh_block_geometry* g, BlockSetup& s) {
  int rc = measure_blocks(op, g, s);
  if (rc) return rc;
  if (g->points_per_cloud <= 0) {
    if (g->table_dev == nullptr) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: ragged clouds need a device table", op);
    s.map.table = reinterpret_cast<const BlockCloud*>(g->table_dev);
  }
  if (!g->node_aabbs || !g->sorted_indices)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL input pointer", op);
  const PlanSizes p = plan_sizes(s, g);
  const size_t need = plan_total(p);
  if (g->plan == nullptr || g->plan_bytes < need)
    return blocks_fail(TBVH_ERR_WORKSPACE, "%s: plan of %zu bytes is smaller than the required %zu", op, g->plan_bytes,
                       need);
  if (uintptr_t(g->plan) % 16 != 0)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: the plan must lie on a multiple of 16 bytes", op);
  char* at = static_cast<char*>(g->plan);
  s.plan.query_row = reinterpret_cast<int*>(at);
  at += p.rows;
  s.plan.query_point = reinterpret_cast<float*>(at);
  at += p.points;
  s.plan.tile_count = reinterpret_cast<int*>(at);
  at += p.count;
  s.plan.entries = reinterpret_cast<uint2*>(at);
  at += p.entries;
  if (g->backward) {
    s.plan.query_begin = reinterpret_cast<int64_t*>(at);
    at += p.begin;
    s.plan.list = reinterpret_cast<uint32_t*>(at);
    at += p.list;
    s.plan.entry_begin = reinterpret_cast<int64_t*>(at);
    at += p.begin;
    s.plan.entry_count = reinterpret_cast<int*>(at);
    at += p.counts;
    s.plan.query_count = reinterpret_cast<int*>(at);
    at += p.counts;
    s.plan.unsorted = reinterpret_cast<uint2*>(at);
  }
  if (g->device >= 0) {
    int cur = -1;
    if (cudaGetDevice(&cur) != cudaSuccess || cur != g->device) {
      const cudaError_t e = cudaSetDevice(g->device);
      if (e != cudaSuccess) return blocks_cuda_fail(e, op);
    }
  }
  return TBVH_OK;
}

namespace {

struct SelectArgs {
  BlockMap map;
  BlockPlan plan;
  const float* aabbs;
  const float* queries;
  const int64_t* order;  // nullable
  bool ordered;          // the plan's query rows are set (k_order_queries)
  int64_t* out_blocks;
  float* out_dist;
  int num;
  unsigned* status;
};

constexpr int kSelectStack = 44;  // <= 3 more nodes per two levels, 25 levels at most
// The tree is cut this many levels above the blocks: the up to 16 blocks below a
// node there are a bunch, scored together.
constexpr int kBunchLevels = 4;
constexpr int kBunch = 1 << kBunchLevels;

template <int D>
struct Box {
  float lo[D], hi[D];
};

template <int D>
__device__ __forceinline__ Box<D> load_box(const float* rows, int64_t row) {
  Box<D> b;
  const float2* p = reinterpret_cast<const float2*>(rows + row * (2 * D));
  if constexpr (D == 3) {
    const float2 u = __ldg(p), v = __ldg(p + 1), w = __ldg(p + 2);
    b.lo[0] = u.x; b.lo[1] = u.y; b.lo[2] = v.x;
    b.hi[0] = v.y; b.hi[1] = w.x; b.hi[2] = w.y;
  } else {
    const float2 u = __ldg(p), v = __ldg(p + 1);
    b.lo[0] = u.x; b.lo[1] = u.y;
    b.hi[0] = v.x; b.hi[1] = v.y;
  }
  return b;
}

template <int D>
__device__ __forceinline__ float box_score(const float* q, const Box<D>& b) {
  float s = 0.0f;
#pragma unroll
  for (int a = 0; a < D; ++a) {
    const float gap = fmaxf(__fsub_rn(b.lo[a], q[a]), fmaxf(__fsub_rn(q[a], b.hi[a]), 0.0f));
    const float sq = __fmul_rn(gap, gap);
    s = a == 0 ? sq : __fadd_rn(s, sq);
  }
  return s;
}

__device__ __forceinline__ uint64_t score_key(float s, uint32_t block) {
  return (uint64_t(__float_as_uint(s)) << 32) | block;
}

// Order of the queries of small clouds: one thread block a cloud, a radix sort of
// their Morton codes (24 bits, within the cloud's box: tiles then begin where blocks
// do), in registers and shared memory. Only which queries share a tile hangs on it.
// One launch in place of the six of the sort over all clouds, which their latency
// bounds there; bound by issue on the few SMs that it runs on. A whole selection of
// 8 blocks, this order / that sort: 2,000 queries 30 / 66 us, 10,000 72 / 88, 16,384
// 89 / 94, 64 x 16,384 367 / 458, 300 x 1,000 56 / 127. Equal digits of a warp are
// found by eight ballots; match instructions took 1.2 times as long.
constexpr int kOrderQueriesThreads = 1024;
constexpr int kSmallQueries = 16 * kOrderQueriesThreads;
static_assert(kSmallQueries == TBVH_SMALL_QUERIES, "as documented");

__host__ __device__ constexpr size_t order_queries_smem(int items) {
  return size_t(items) * kOrderQueriesThreads * 6 + kOrderQueriesThreads / 32 * 256 * 4;
}

template <int D, int ITEMS>
__global__ void __launch_bounds__(kOrderQueriesThreads) k_order_queries(BlockMap map, const float* aabbs,
                                                                       const float* queries, int* query_row) {
  constexpr int WARPS = kOrderQueriesThreads / 32, COUNT = ITEMS * kOrderQueriesThreads;
  extern __shared__ __align__(16) char smem[];
  uint32_t* s_key = reinterpret_cast<uint32_t*>(smem);           // [COUNT]
  uint32_t* s_count = s_key + COUNT;                             // [WARPS][256]
  uint16_t* s_val = reinterpret_cast<uint16_t*>(s_count + WARPS * 256);  // [COUNT]
  __shared__ uint32_t s_base[256], s_warp[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const BlockCloud c = map.of_cloud(blockIdx.x);
  const int m = int(c.m);
  const float* q = queries + c.q0 * D;

  const Box<D> scene = load_box<D>(aabbs, c.row0);
  constexpr int BINS = D == 3 ? 256 : 4096;  // an axis
  float scale[D];
#pragma unroll
  for (int x = 0; x < D; ++x) scale[x] = scene.hi[x] > scene.lo[x] ? float(BINS) / (scene.hi[x] - scene.lo[x]) : 0.0f;
  auto bin = [&](float v, int x) { return uint32_t(fminf(fmaxf((v - scene.lo[x]) * scale[x], 0.0f), float(BINS - 1))); };
  // Element j of a lane: place warp * 32 * ITEMS + j * 32 + lane. Places past the
  // cloud's queries have the highest key and, the sort being stable, stay last.
  const int first = warp * 32 * ITEMS + lane;
  uint32_t key[ITEMS];
  uint32_t val[ITEMS];  // query, and in the upper half its rank among its warp's equal digits
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int i = first + j * 32;
    key[j] = 0xffffffu;
    if (i < m) {
      const float* v = q + int64_t(i) * D;
      if constexpr (D == 3)
        key[j] = spread_bits3(bin(__ldg(v), 0)) | spread_bits3(bin(__ldg(v + 1), 1)) << 1 |
                 spread_bits3(bin(__ldg(v + 2), 2)) << 2;
      else
        key[j] = spread_bits2(bin(__ldg(v), 0)) | spread_bits2(bin(__ldg(v + 1), 1)) << 1;
    }
    val[j] = uint32_t(i);
  }
  uint32_t* mine = s_count + warp * 256;
#pragma unroll 1
  for (int shift = 0; shift < 24; shift += 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) mine[i * 32 + lane] = 0;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const uint32_t digit = key[j] >> shift & 255u;
      unsigned peers = kFullMask;  // lanes with the same digit
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const unsigned set = __ballot_sync(kFullMask, digit >> b & 1u);
        peers &= (digit >> b & 1u) ? set : ~set;
      }
      const uint32_t below = __popc(peers & ((1u << lane) - 1));
      const uint32_t before = mine[digit];
      __syncwarp();
      if (below == 0) mine[digit] = before + __popc(peers);
      __syncwarp();
      val[j] = (val[j] & 0xffffu) | (before + below) << 16;
    }
    __syncthreads();
    // Every digit's first place, and its warps' places behind that.
    uint32_t total = 0, x = 0;
    if (tid < 256) {
      for (int w = 0; w < WARPS; ++w) {
        const uint32_t n = s_count[w * 256 + tid];
        s_count[w * 256 + tid] = total;
        total += n;
      }
      x = total;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(kFullMask, x, d);
        if (lane >= d) x += y;
      }
      if (lane == 31) s_warp[warp] = x;
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t base = x - total;
      for (int w = 0; w < warp; ++w) base += s_warp[w];
      s_base[tid] = base;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const uint32_t digit = key[j] >> shift & 255u;
      const uint32_t place = s_base[digit] + mine[digit] + (val[j] >> 16);
      s_key[place] = key[j];
      s_val[place] = uint16_t(val[j]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      key[j] = s_key[first + j * 32];
      val[j] = s_val[first + j * 32];
    }
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    if (first + j * 32 < m) query_row[c.t0 * kTileQueries + first + j * 32] = int(c.q0 + val[j]);
}

// Inserts x into ascending keys from the top, kInsertGroup slots at a time: below
// the group where no lane's x belongs nothing moves, and candidates come with
// ascending bounds, so most belong near the end (16 x 65,536 points, 16 blocks:
// 1.13 ms for groups of four, 1.12 of two, 1.18 of eight, 1.29 for all 16; 32
// blocks of 4 x 65,536: 605, 643, 628 and 796 us).
constexpr int kInsertGroup = 4;

template <int CAP, int HI>
__device__ __forceinline__ void insert_key(uint64_t (&key)[CAP], uint64_t x) {
  constexpr int LO = HI > kInsertGroup ? HI - kInsertGroup : 0;
#pragma unroll
  for (int i = HI - 1; i > LO; --i) key[i] = x < key[i - 1] ? key[i - 1] : (x < key[i] ? x : key[i]);
  if constexpr (LO == 0) {
    key[0] = x < key[0] ? x : key[0];
  } else if (x < key[LO - 1]) {
    key[LO] = key[LO - 1];
    insert_key<CAP, LO>(key, x);
  } else {
    key[LO] = x < key[LO] ? x : key[LO];
  }
}

// Ascending: the lowest CAP of this lane's keys and of `other`, both ascending.
template <int CAP>
__device__ __forceinline__ void merge_keys(uint64_t (&key)[CAP], const uint64_t* other) {
#pragma unroll
  for (int i = 0; i < CAP; ++i) {  // the lower of each pair from opposite ends: a bitonic sequence
    const uint64_t x = other[CAP - 1 - i];
    key[i] = x < key[i] ? x : key[i];
  }
#pragma unroll
  for (int d = CAP / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < CAP; ++i)
      if ((i & d) == 0) {
        const uint64_t a = key[i], b = key[i + d];
        key[i] = a < b ? a : b;
        key[i + d] = a < b ? b : a;
      }
}

// WARPS warps a tile: one where tiles fill the GPU, four where they do not and the
// time is one warp's. Each then takes every fourth bunch of the tree (below) into
// lists of its own, which are merged at the end; all prune by the least of a query's
// k-th keys, which the k-th best of all cannot exceed. Whole calls of 8 (32) blocks,
// one warp / four: 22 tiles 168 / 101 us (353 / 208), 313 tiles 75 / 62 (118 / 111),
// 512 tiles 91 / 81 (152 / 148), 1,024 tiles 98 / 91 (173 / 236).
//
// A warp walks the tree as a packet, two levels a step: the
// (up to four) grandchildren of a node are scored by every lane, those that some
// lane admits are pushed, the one nearest to most lanes last. A popped node is
// scored again against the meanwhile lower k-th keys. At a bunch each of 16
// lanes loads one block's box and scores it against the box of the tile's
// queries, a lower bound for all of them; the boxes go to shared memory in
// ascending order of that bound, so that near blocks enter the lists first, few
// are displaced again, and the scan ends at the first block no query can want.
// Bound by issue: an insertion shifts a list of 64-bit keys in registers (16 x
// 65,536 queries, 16 blocks: 0.85 of the 1.05 ms of the call with its lists, issue
// slots 73 % and the integer pipe 64 % busy, DRAM 3 %). One block at a time instead of
// bunches in order took 1.2 times as long.
template <int D, int CAP, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) k_select(SelectArgs a) {
  __shared__ uint32_t s_stacks[WARPS][kSelectStack];
  __shared__ int64_t s_rows[WARPS][32];
  __shared__ uint64_t s_keys[WARPS * 32 * CAP];
  __shared__ int64_t s_query[32];
  __shared__ float4 s_los[WARPS][kBunch], s_his[WARPS][kBunch];  // w: lower bound, block
  __shared__ unsigned long long s_bound[32];                     // WARPS > 1: least k-th key of each query
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* s_stack = s_stacks[warp];
  int64_t* s_row = s_rows[warp];
  float4 *s_lo = s_los[warp], *s_hi = s_his[warp];
  const int64_t tile = blockIdx.x;
  const BlockCloud c = a.map.of_tile(tile);
  const int64_t pos = (tile - c.t0) * kTileQueries + lane;
  const int leaf_level = ceil_log2_i64(c.n);
  const int last = leaf_level > kBlockLevels ? leaf_level - kBlockLevels : 0;  // level of the blocks

  // First node row of every level: exclusive sum of the level counts.
  {
    const int64_t count = lane <= leaf_level ? level_count(c.n, leaf_level, lane) : 0;
    int64_t x = count;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(kFullMask, x, d);
      if (lane >= d) x += y;
    }
    s_row[lane] = c.row0 + x - count;
  }

  bool active = pos < c.m;
  int64_t query = -1;
  if (active) {
    const int64_t local = a.ordered ? a.plan.query_row[tile * kTileQueries + lane] - c.q0
                          : a.order ? a.order[c.q0 + pos]
                                    : pos;
    if (local < 0 || local >= c.m) {
      if (a.status) atomicOr(a.status, kDevErrBadIndex);
      active = false;
    } else {
      query = c.q0 + local;
    }
  }
  if constexpr (WARPS > 1) __syncthreads();  // all have read the row
  if (warp == 0) {
    s_query[lane] = query;
    a.plan.query_row[tile * kTileQueries + lane] = int(query);
  }
  float q[D];
  bool searching = active;
#pragma unroll
  for (int x = 0; x < D; ++x) {
    q[x] = active ? a.queries[query * D + x] : 0.0f;
    searching = searching && q[x] == q[x];  // a NaN query selects nothing
  }
#pragma unroll
  for (int x = 0; x < 3; ++x)
    if (warp == 0) a.plan.query_point[(tile * 3 + x) * kTileQueries + lane] = x < D ? q[x < D ? x : 0] : 0.0f;
  // Ascending keys; the first CAP - num slots hold 0 and stay, so the last slot
  // is the num-th best. Admission: key < last slot.
  const uint64_t empty = uint64_t(__float_as_uint(kFar)) << 32;
  uint64_t key[CAP];
#pragma unroll
  for (int i = 0; i < CAP; ++i) key[i] = i < CAP - a.num ? 0 : empty;
  if (!searching) {
#pragma unroll
    for (int i = 0; i < CAP; ++i) key[i] = empty;
  }
  // A lane that does not search admits nothing: its bound is 0.
  uint64_t bound = searching ? empty : 0;
  if constexpr (WARPS > 1) {
    if (warp == 0) s_bound[lane] = bound;
    __syncthreads();
  }
  __syncwarp();

  auto insert = [&](uint64_t x) {
    if (x < bound) {
      insert_key<CAP, CAP>(key, x);
      bound = key[CAP - 1] < bound ? key[CAP - 1] : bound;
    }
  };

  // The box of the tile's queries.
  float q_lo[D], q_hi[D];
#pragma unroll
  for (int x = 0; x < D; ++x) {
    q_lo[x] = searching ? q[x] : INFINITY;
    q_hi[x] = searching ? q[x] : -INFINITY;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      q_lo[x] = fminf(q_lo[x], __shfl_xor_sync(kFullMask, q_lo[x], d));
      q_hi[x] = fmaxf(q_hi[x], __shfl_xor_sync(kFullMask, q_hi[x], d));
    }
  }
  // The largest k-th score of any lane.
  auto worst = [&]() { return __uint_as_float(__reduce_max_sync(kFullMask, uint32_t(bound >> 32))); };

  const int bunch_level = last > kBunchLevels ? last - kBunchLevels : 0;
  const int below = last - bunch_level;  // levels from a bunch's node to its blocks
  auto scan_bunch = [&](uint32_t node) {
    const uint32_t base = node << below;
    const int64_t there = level_count(c.n, leaf_level, last) - base;
    const int blocks = there < (1 << below) ? int(there) : 1 << below;
    float least = INFINITY;
    Box<D> box{};
    if (lane < blocks) {
      box = load_box<D>(a.aabbs, s_row[last] + base + lane);
      float sum = 0.0f;
#pragma unroll
      for (int x = 0; x < D; ++x) {
        const float gap = fmaxf(__fsub_rn(box.lo[x], q_hi[x]), fmaxf(__fsub_rn(q_lo[x], box.hi[x]), 0.0f));
        const float sq = __fmul_rn(gap, gap);
        sum = x == 0 ? sq : __fadd_rn(sum, sq);
      }
      least = sum == sum ? sum : 0.0f;
    }
    // Place in ascending order of the bound (the lower block first among equals).
    int place = 0;
#pragma unroll
    for (int k = 0; k < kBunch; ++k) {
      const float other = __shfl_sync(kFullMask, least, k);
      place += other < least || (other == least && k < lane);
    }
    __syncwarp();
    if (lane < blocks) {
      s_lo[place] = make_float4(box.lo[0], box.lo[1], D == 3 ? box.lo[D - 1] : 0.0f, least);
      s_hi[place] = make_float4(box.hi[0], box.hi[1], D == 3 ? box.hi[D - 1] : 0.0f, __uint_as_float(base + lane));
    }
    __syncwarp();
    if constexpr (WARPS > 1) {  // the other warps' progress
      const uint64_t shared = *static_cast<volatile unsigned long long*>(s_bound + lane);
      bound = shared < bound ? shared : bound;
    }
    float reach = worst();
    for (int k = 0; k < blocks; ++k) {
      const float4 lo = s_lo[k], hi = s_hi[k];
      if (lo.w > reach) break;
      Box<D> b;
      b.lo[0] = lo.x, b.lo[1] = lo.y, b.hi[0] = hi.x, b.hi[1] = hi.y;
      if constexpr (D == 3) b.lo[2] = lo.z, b.hi[2] = hi.z;
      const uint64_t x = score_key(box_score<D>(q, b), __float_as_uint(hi.w));
      if (__any_sync(kFullMask, x < bound)) {
        insert(x);
        reach = worst();
      }
    }
    if constexpr (WARPS > 1) atomicMin(s_bound + lane, static_cast<unsigned long long>(bound));
  };

  int depth = 0;
  if (bunch_level == 0) {
    if (warp == 0) scan_bunch(0);
  } else {
    if (lane == 0) s_stack[0] = 0;
    depth = 1;
  }
  __syncwarp();
  bool fresh = true;  // the root needs no second look
  while (depth > 0) {
    --depth;
    const uint32_t node = s_stack[depth];
    __syncwarp();
    const int level = int(node >> 27);
    const uint32_t j = node & 0x7ffffffu;
    if (!fresh) {
      const float s = box_score<D>(q, load_box<D>(a.aabbs, s_row[level] + j));
      if (!__any_sync(kFullMask, score_key(s, j << (last - level)) < bound)) continue;
    }
    fresh = false;
    if (level == bunch_level) {
      scan_bunch(j);
      continue;
    }
    const int step = bunch_level - level >= 2 ? 2 : 1;
    const int child_level = level + step;
    const uint32_t base = j << step;
    const int64_t there = level_count(c.n, leaf_level, child_level) - base;
    const int children = there < (1 << step) ? int(there) : (1 << step);
    float score[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      score[k] = k < children ? box_score<D>(q, load_box<D>(a.aabbs, s_row[child_level] + base + k)) : kFar;
    // Every lane votes for its nearest child that it admits.
    int nearest = -1;
    float least = kFar;
    unsigned admitted = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool here = WARPS == 1 || child_level < bunch_level || int(base + k) % WARPS == warp;
      const bool ok = here && k < children && score_key(score[k], (base + k) << (last - child_level)) < bound;
      if (__any_sync(kFullMask, ok)) admitted |= 1u << k;
      if (ok && score[k] < least) {
        least = score[k];
        nearest = k;
      }
    }
    int votes[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      votes[k] = (admitted >> k & 1u) ? __popc(__ballot_sync(kFullMask, nearest == k)) : -1;
    if (depth + 4 > kSelectStack) {
      if (a.status && lane == 0) atomicOr(a.status, kDevErrStackOverflow);
      break;
    }
    // Fewest votes first; among equals the higher child first (popped later).
#pragma unroll
    for (int round = 0; round < 4; ++round) {
      int pick = -1;
#pragma unroll
      for (int k = 3; k >= 0; --k)
        if (votes[k] >= 0 && (pick < 0 || votes[k] < (pick == 3 ? votes[3] : pick == 2 ? votes[2] : votes[1]))) pick = k;
      if (pick >= 0) {
        if (lane == 0) s_stack[depth] = (uint32_t(child_level) << 27) | (base + pick);
        ++depth;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k == pick) votes[k] = -1;
      }
    }
    __syncwarp();
  }

  uint64_t* own = s_keys + threadIdx.x * CAP;
#pragma unroll
  for (int i = 0; i < CAP; ++i) own[i] = key[i];
  if constexpr (WARPS > 1) {
    // The slots in use to the front: lists that ascend throughout. Then warp w takes in
    // the lists of warp w + 1, and so on by doubles.
#pragma unroll
    for (int i = 0; i < CAP; ++i) key[i] = i < a.num ? own[CAP - a.num + i] : ~uint64_t(0);
#pragma unroll
    for (int d = 1; d < WARPS; d *= 2) {
#pragma unroll
      for (int i = 0; i < CAP; ++i) own[i] = key[i];
      __syncthreads();
      if (warp % (2 * d) == 0) merge_keys(key, own + d * 32 * CAP);
      __syncthreads();
    }
    if (warp != 0) return;
#pragma unroll
    for (int i = 0; i < CAP; ++i)
      if (i < a.num) own[CAP - a.num + i] = key[i];
#pragma unroll
    for (int i = 0; i < CAP; ++i) key[i] = i < CAP - a.num ? 0 : own[i];
  }
  __syncwarp();
  // Rows of the result, written a row at a time: slot s of lane r by lane s.
  {
    int r = lane / a.num, slot = lane % a.num;
    const int dr = 32 / a.num, ds = 32 % a.num;
    for (int i = lane; i < 32 * a.num; i += 32) {
      const int64_t row = s_query[r];
      if (row >= 0) {
        const uint64_t k = s_keys[r * CAP + CAP - a.num + slot];
        const bool none = k >= empty;
        a.out_blocks[row * a.num + slot] = none ? -1 : int64_t(uint32_t(k));
        a.out_dist[row * a.num + slot] = none ? kFar : __uint_as_float(uint32_t(k >> 32));
      }
      r += dr;
      slot += ds;
      if (slot >= a.num) {
        slot -= a.num;
        ++r;
      }
    }
  }

  // Union of the lanes' blocks in ascending order: each round takes the least
  // block above the previous one.
  uint32_t id[CAP];
#pragma unroll
  for (int i = 0; i < CAP; ++i) {
    const bool real = searching && i >= CAP - a.num && key[i] < empty;
    id[i] = real ? uint32_t(key[i]) + 1 : 0;  // 0: none
  }
  uint32_t done = 0;
  int count = 0;
  uint2* entries = a.plan.entries + tile * a.plan.capacity;
  while (count < a.plan.capacity) {
    uint32_t next = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < CAP; ++i) next = id[i] > done && id[i] < next ? id[i] : next;
    const uint32_t least = __reduce_min_sync(kFullMask, next);
    if (least == 0xffffffffu) break;
    const unsigned mask = __ballot_sync(kFullMask, next == least);
    if (lane == 0) {
      entries[count] = make_uint2(least - 1, mask);
      if (a.plan.entry_count) {
        atomicAdd(a.plan.entry_count + c.b0 + (least - 1), 1);
        atomicAdd(a.plan.query_count + c.b0 + (least - 1), __popc(mask));
      }
    }
    ++count;
    done = least;
  }
  if (lane == 0) a.plan.tile_count[tile] = count;
}

// Exclusive sums of the blocks' counts: of entries (thread block 0, which also
// sets the counts to 0 as fill cursors) and of queries (thread block 1). Eight
// values a thread and step.
__global__ void __launch_bounds__(1024) k_block_begin(BlockPlan plan, int64_t blocks) {
  __shared__ int64_t s_warp[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* counts = blockIdx.x == 0 ? plan.entry_count : plan.query_count;
  int64_t* begin = blockIdx.x == 0 ? plan.entry_begin : plan.query_begin;
  int64_t carry = 0;
  for (int64_t at = 0; at < blocks; at += 8 * 1024) {
    int64_t sum = 0;
    int v[8] = {};
    const int64_t mine = at + tid * 8;
    const bool full = mine + 8 <= blocks;
    if (full) {
      *reinterpret_cast<int4*>(v) = *reinterpret_cast<const int4*>(counts + mine);
      *reinterpret_cast<int4*>(v + 4) = *reinterpret_cast<const int4*>(counts + mine + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mine + i < blocks ? counts[mine + i] : 0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[i];
    int64_t x = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(kFullMask, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int64_t before = carry, total = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += s_warp[w];
      total += s_warp[w];
    }
    before += x - sum;
    if (full) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        *reinterpret_cast<longlong2*>(begin + mine + i) = make_longlong2(before, before + v[i]);
        before += v[i] + v[i + 1];
      }
      if (blockIdx.x == 0)
        for (int i = 0; i < 8; i += 4) *reinterpret_cast<int4*>(counts + mine + i) = make_int4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (mine + i < blocks) {
          begin[mine + i] = before;
          if (blockIdx.x == 0) counts[mine + i] = 0;
        }
        before += v[i];
      }
    }
    carry += total;
    __syncthreads();
  }
  if (tid == 0) begin[blocks] = carry;
}

// Every tile's entries into their blocks' runs, in order of arrival (the next
// kernel puts them in order). One warp a tile.
__global__ void __launch_bounds__(128) k_block_fill(BlockMap map, BlockPlan plan) {
  const int64_t tile = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (tile >= map.num_tiles) return;
  const BlockCloud c = map.of_tile(tile);
  const uint2* e = plan.entries + tile * plan.capacity;
  const int count = plan.tile_count[tile];
  for (int i = threadIdx.x & 31; i < count; i += 32) {
    const int64_t block = c.b0 + e[i].x;
    const int64_t at = plan.entry_begin[block] + atomicAdd(plan.entry_count + block, 1);
    plan.unsorted[at] = make_uint2(uint32_t(tile), e[i].y);
  }
}

// Every block's queries in ascending order, whatever order its entries arrived
// in. An entry's first place is the number of queries in entries of lower
// tiles: by comparison in shared memory for short runs; for long ones by a
// bitmap of the queries of a window of tiles (a tile's word is its mask), whose
// words are counted.
constexpr int kOrderThreads = 128;
constexpr int kOrderShort = 512;
constexpr int kOrderWords = 2048;

__device__ __forceinline__ void write_slots(uint32_t* out, uint32_t tile, uint32_t mask) {
  for (; mask != 0; mask &= mask - 1) *out++ = tile * kTileQueries + (__ffs(mask) - 1);
}

__global__ void __launch_bounds__(kOrderThreads) k_block_order(BlockMap map, BlockPlan plan) {
  __shared__ uint2 s_entry[kOrderShort];
  __shared__ uint32_t s_bits[kOrderWords];
  __shared__ int s_warp[kOrderThreads / 32];
  const int tid = threadIdx.x;
  const int64_t block = blockIdx.x;
  const int64_t begin = plan.entry_begin[block];
  const int64_t count = plan.entry_begin[block + 1] - begin;
  const uint2* in = plan.unsorted + begin;
  uint32_t* out = plan.list + plan.query_begin[block];
  if (count <= kOrderShort) {
    for (int i = tid; i < count; i += kOrderThreads) s_entry[i] = in[i];
    __syncthreads();
    // Through shared memory where the list fits: whole lines to memory instead of words.
    const int64_t queries = plan.query_begin[block + 1] - plan.query_begin[block];
    const bool fits = queries <= kOrderWords;
    for (int i = tid; i < count; i += kOrderThreads) {
      const uint2 mine = s_entry[i];
      int before = 0;
      for (int k = 0; k < count; ++k) {
        const uint2 e = s_entry[k];
        before += e.x < mine.x ? __popc(e.y) : 0;
      }
      write_slots((fits ? s_bits : out) + before, mine.x, mine.y);
    }
    if (!fits) return;
    __syncthreads();
    for (int i = tid; i < queries; i += kOrderThreads) out[i] = s_bits[i];
    return;
  }
  const BlockCloud c = map.of_block(block);
  const int64_t tiles = tiles_of(c.m);
  int64_t placed = 0;
  for (int64_t first = 0; first < tiles; first += kOrderWords) {
    for (int w = tid; w < kOrderWords; w += kOrderThreads) s_bits[w] = 0;
    __syncthreads();
    for (int64_t i = tid; i < count; i += kOrderThreads) {
      const int64_t t = int64_t(in[i].x) - c.t0 - first;
      if (t >= 0 && t < kOrderWords) s_bits[t] = in[i].y;
    }
    __syncthreads();
    // Exclusive counts; thread t owns words [t * per, (t + 1) * per).
    constexpr int per = kOrderWords / kOrderThreads;
    int sum = 0;
#pragma unroll
    for (int i = 0; i < per; ++i) sum += __popc(s_bits[tid * per + i]);
    int x = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(kFullMask, x, d);
      if ((tid & 31) >= d) x += y;
    }
    if ((tid & 31) == 31) s_warp[tid >> 5] = x;
    __syncthreads();
    int before = x - sum, total = 0;
#pragma unroll
    for (int w = 0; w < kOrderThreads / 32; ++w) {
      if (w < (tid >> 5)) before += s_warp[w];
      total += s_warp[w];
    }
    for (int i = 0; i < per; ++i) {
      const uint32_t mask = s_bits[tid * per + i];
      write_slots(out + placed + before, uint32_t(c.t0 + first + tid * per + i), mask);
      before += __popc(mask);
    }
    placed += total;
    __syncthreads();
  }
}

constexpr int64_t kFewTiles = 4 * 148;  // below four tiles an SM a tile has four warps

template <int D, int ITEMS>
cudaError_t launch_order(const SelectArgs& a, cudaStream_t stream) {
  constexpr size_t smem = order_queries_smem(ITEMS);
  if (smem > 48 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(k_order_queries<D, ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
  }
  k_order_queries<D, ITEMS><<<unsigned(a.map.num_clouds), kOrderQueriesThreads, smem, stream>>>(a.map, a.aabbs, a.queries,
                                                                                               a.plan.query_row);
  count_launches(1);
  return cudaGetLastError();
}

template <int D>
cudaError_t launch_select(SelectArgs a, int64_t most_queries, int64_t most_blocks, cudaStream_t stream) {
  a.ordered = a.order == nullptr && most_queries > kTileQueries && most_queries <= kSmallQueries;
  if (a.ordered) {
    const int items = int((most_queries + kOrderQueriesThreads - 1) / kOrderQueriesThreads);
    const cudaError_t e = items == 1   ? launch_order<D, 1>(a, stream)
                          : items <= 4 ? launch_order<D, 4>(a, stream)
                          : items <= 8 ? launch_order<D, 8>(a, stream)
                          : items <= 12 ? launch_order<D, 12>(a, stream)
                                        : launch_order<D, 16>(a, stream);
    if (e != cudaSuccess) return e;
  }
  const unsigned grid = unsigned(a.map.num_tiles);
  const bool few = a.map.num_tiles < kFewTiles && most_blocks > kBunch;
  auto go = [&](auto cap) {
    constexpr int CAP = decltype(cap)::value;
    if (few) k_select<D, CAP, 4><<<grid, 128, 0, stream>>>(a);
    else k_select<D, CAP, 1><<<grid, 32, 0, stream>>>(a);
  };
  if (a.num <= 4) go(std::integral_constant<int, 4>{});
  else if (a.num <= 8) go(std::integral_constant<int, 8>{});
  else if (a.num <= 16) go(std::integral_constant<int, 16>{});
  else go(std::integral_constant<int, 32>{});
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace
}  // namespace tbvh

extern "C" {

int tbvh_block_table(int64_t num_clouds, const int64_t* point_offsets, const int64_t* query_offsets,
                     int64_t* table_out) {
  const char* op = "block_table";
  if (num_clouds < 1 || !point_offsets || !query_offsets || !table_out)
    return tbvh::blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL pointer or no clouds", op);
  if (point_offsets[0] != 0 || query_offsets[0] != 0)
    return tbvh::blocks_fail(TBVH_ERR_BAD_ARG, "%s: offsets must start at 0", op);
  auto* t = reinterpret_cast<tbvh::BlockCloud*>(table_out);
  tbvh::BlockCloud c{};
  for (int64_t b = 0; b < num_clouds; ++b) {
    c.n = point_offsets[b + 1] - point_offsets[b];
    c.m = query_offsets[b + 1] - query_offsets[b];
    if (c.n < 1) return tbvh::blocks_fail(TBVH_ERR_BAD_ARG, "%s: offsets must be strictly increasing", op);
    if (c.m < 0) return tbvh::blocks_fail(TBVH_ERR_BAD_ARG, "%s: query offsets must not decrease", op);
    t[b] = c;
    c.p0 += c.n;
    c.row0 += tbvh::real_node_count(c.n);
    c.q0 += c.m;
    c.t0 += tbvh::tiles_of(c.m);
    c.b0 += tbvh::blocks_of(c.n);
  }
  return TBVH_OK;
}

size_t tbvh_block_plan_size(const tbvh_block_geometry* g) {
  tbvh::BlockSetup s;
  if (tbvh::measure_blocks("select_blocks", g, s)) return 0;
  return tbvh::plan_total(tbvh::plan_sizes(s, g));
}

int tbvh_select_blocks(const tbvh_block_geometry* g, int64_t* out_blocks, float* out_distances, void* stream) {
  using namespace tbvh;
  const char* op = "select_blocks";
  BlockSetup s;
  int rc = setup_blocks(op, g, s);
  if (rc) return rc;
  if (s.total_queries > 0 && (!g->query_points || !out_blocks || !out_distances))
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL query or output pointer", op);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (s.plan.entry_count)  // both counts, side by side
    e = cudaMemsetAsync(s.plan.entry_count, 0,
                        size_t(reinterpret_cast<char*>(s.plan.unsorted) - reinterpret_cast<char*>(s.plan.entry_count)), st);
  if (e == cudaSuccess && s.map.num_tiles > 0) {
    SelectArgs a{};
    a.map = s.map;
    a.plan = s.plan;
    a.aabbs = g->node_aabbs;
    a.queries = g->query_points;
    a.order = g->order;
    a.out_blocks = out_blocks;
    a.out_dist = out_distances;
    a.num = g->num_blocks;
    a.status = device_status_ptr();
    e = g->dim == 3 ? launch_select<3>(a, s.most_queries, s.most_blocks, st)
                    : launch_select<2>(a, s.most_queries, s.most_blocks, st);
  }
  if (e == cudaSuccess && s.plan.entry_count) {
    k_block_begin<<<2, 1024, 0, st>>>(s.plan, s.map.num_blocks);
    if (s.map.num_tiles > 0) k_block_fill<<<unsigned((s.map.num_tiles + 3) / 4), 128, 0, st>>>(s.map, s.plan);
    k_block_order<<<unsigned(s.map.num_blocks), kOrderThreads, 0, st>>>(s.map, s.plan);
    count_launches(s.map.num_tiles > 0 ? 3 : 2);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? TBVH_OK : blocks_cuda_fail(e, op);
}

}  // extern "C"
