// C entries of block attention: argument checks, launch plans, and the small
// kernels around the two backward passes.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "tbvh_attend_q.cuh"
#include "tbvh_kernels.h"

namespace tbvh {
namespace {

// The largest finite |x| as float bits, which order like unsigned numbers.
__device__ __forceinline__ unsigned largest_bits(unsigned most, float x) {
  x = fabsf(x);
  return x <= FLT_MAX ? max(most, __float_as_uint(x)) : most;
}

// The block's largest into *most (a maximum has no order of its own).
__device__ void join_largest(unsigned big, unsigned* most) {
  __shared__ unsigned s_most[8];
  big = __reduce_max_sync(kFullMask, big);
  if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = big;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) big = max(big, s_most[w]);
    atomicMax(most, big);
  }
}

// Largest finite |x| of `count` values; WIDE: read eight at a time.
template <bool WIDE>
__global__ void __launch_bounds__(256) k_largest(const __half* x, int64_t count, unsigned* most) {
  unsigned big = 0;
  const int64_t first = int64_t(blockIdx.x) * 256 + threadIdx.x, step = int64_t(gridDim.x) * 256;
  if constexpr (WIDE) {
    for (int64_t i = first; i < count / 8; i += step) {
      const uint4 w = reinterpret_cast<const uint4*>(x)[i];
#pragma unroll
      for (const unsigned two : {w.x, w.y, w.z, w.w}) {
        const float2 y = Frag<__half>::unpack(two);
        big = largest_bits(largest_bits(big, y.x), y.y);
      }
    }
  } else {
    for (int64_t i = first; i < count; i += step) big = largest_bits(big, __half2float(x[i]));
  }
  join_largest(big, most);
}

cudaError_t run_largest(const __half* x, int64_t count, unsigned* most, cudaStream_t stream) {
  const bool wide = count % 8 == 0 && uintptr_t(x) % 16 == 0;
  const int64_t blocks = (count / (wide ? 8 : 1) + 255) / 256;
  const unsigned grid = unsigned(blocks < 1 ? 1 : blocks > 1184 ? 1184 : blocks);
  if (wide) k_largest<true><<<grid, 256, 0, stream>>>(x, count, most);
  else k_largest<false><<<grid, 256, 0, stream>>>(x, count, most);
  count_launches(1);
  return cudaGetLastError();
}

// delta[row][head] = <grad_out, out>, and for float16 the largest finite |grad_out|.
// `lanes` lanes a (row, head), four channels each at a time where FOUR (rows of
// whole 16-byte words), else one. Bound by reading both tensors once.
template <typename T, typename O, bool FOUR>
__global__ void __launch_bounds__(256) k_delta(const T* grad, const O* out, float* delta, unsigned* most, int64_t rows,
                                               int channels, int lanes) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t(blockIdx.x) * 256 + threadIdx.x) / lanes;
  const int part = lane & (lanes - 1);
  unsigned big = 0;
  float sum = 0.0f;
  if (row < rows) {
    const T* g = grad + row * channels;
    const O* o = out + row * channels;
    constexpr int W = FOUR ? 4 : 1;
    for (int i = part * W; i < channels; i += lanes * W) {
      T x[W];
      O y[W];
      if constexpr (FOUR) {
        using WordT = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
        using WordO = typename std::conditional<sizeof(O) == 2, uint2, uint4>::type;
        *reinterpret_cast<WordT*>(x) = *reinterpret_cast<const WordT*>(g + i);
        *reinterpret_cast<WordO*>(y) = *reinterpret_cast<const WordO*>(o + i);
      } else {
        x[0] = g[i];
        y[0] = o[i];
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float v = Frag<T>::to_float(x[w]);
        sum = fmaf(v, Frag<O>::to_float(y[w]), sum);
        big = largest_bits(big, v);
      }
    }
  }
  for (int d = lanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(kFullMask, sum, d);
  if (row < rows && part == 0) delta[row] = sum;
  if (most != nullptr) join_largest(big, most);
}

template <typename T>
cudaError_t run_delta(const void* grad, const void* out, const float* exact, float* delta, unsigned* most,
                      int64_t pairs, int channels, cudaStream_t stream) {
  const T* g = static_cast<const T*>(grad);
  const void* o = exact ? static_cast<const void*>(exact) : out;
  const bool four = channels % 4 == 0 && uintptr_t(g) % (4 * sizeof(T)) == 0 &&
                    uintptr_t(o) % (4 * (exact ? sizeof(float) : sizeof(T))) == 0;
  int lanes = 1;
  while (lanes < 32 && lanes * (four ? 4 : 1) < channels) lanes *= 2;
  const unsigned grid = unsigned((pairs * lanes + 255) / 256);
  if (exact) {
    if (four) k_delta<T, float, true><<<grid, 256, 0, stream>>>(g, exact, delta, most, pairs, channels, lanes);
    else k_delta<T, float, false><<<grid, 256, 0, stream>>>(g, exact, delta, most, pairs, channels, lanes);
  } else {
    const T* same = static_cast<const T*>(out);
    if (four) k_delta<T, T, true><<<grid, 256, 0, stream>>>(g, same, delta, most, pairs, channels, lanes);
    else k_delta<T, T, false><<<grid, 256, 0, stream>>>(g, same, delta, most, pairs, channels, lanes);
  }
  count_launches(1);
  return cudaGetLastError();
}

size_t pad256(size_t v) { return (v + 255) / 256 * 256; }

// Splits of the kernels by query tile: enough thread blocks for four an SM when the
// tiles alone are fewer than two, never more than a tile can have entries (training
// passes, float32: 189 thread blocks 564 us, 613 when only fewer than 148 were split;
// 64 of one head of 96 over 12 blocks 811 us, 1,351 as one).
int tile_splits(const BlockSetup& s, const AttendArgs& a) {
  const int64_t blocks = s.map.num_tiles * head_groups(a);
  if (blocks <= 0 || blocks >= 2 * 148) return 1;
  int64_t want = (4 * 148 + blocks - 1) / blocks;
  if (want > s.plan.capacity) want = s.plan.capacity;
  return int(want < 1 ? 1 : want > 32 ? 32 : want);
}

// Heads of a thread block of the query-tile kernels: four (eight warps) share the
// buckets of a bias, two are enough without one (measured at 65,536 queries, 4
// heads of 32 / 64 channels, bf16: with bias 319 / 501 us for four and 364 / 521
// for two; without 242 / 414 and 229 / 357); fewer where two thread blocks would
// not share an SM's memory.
void plan_heads(AttendArgs& a, int size, bool back) {
  const int cp = padded_channels(a.channels);
  const int most = a.buckets > 0 ? 4 : 2;
  int kv = a.group > most ? 1 : most / a.group;
  if (kv > a.kv_heads) kv = a.kv_heads;
  a.kv_cta = kv;
  a.heads_cta = a.group > most ? most : kv * a.group;
  while (a.heads_cta > 1 &&
         query_tile_smem(size, cp, a.kv_cta, a.heads_cta, back, a.buckets > 0, a.buckets).total > 110 * 1024) {
    if (a.kv_cta > 1) {
      --a.kv_cta;
      a.heads_cta = a.kv_cta * a.group;
    } else {
      --a.heads_cta;  // part of a group
    }
  }
}

// Whether every pointer (NULL or not) lies on a multiple of `size`.
template <typename... P>
bool aligned(size_t size, P... pointers) {
  return ((uintptr_t(pointers) % size == 0) && ...);
}

int element_size(int dtype) { return dtype == TBVH_F32 ? 4 : 2; }

int misaligned(const char* op) { return blocks_fail(TBVH_ERR_BAD_ARG, "%s: a pointer is not aligned to its type", op); }

int check_features(const char* op, const tbvh_attend_features* f, bool pointers) {
  if (f == nullptr) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: features are NULL", op);
  if (f->dtype != TBVH_F32 && f->dtype != TBVH_F16 && f->dtype != TBVH_BF16)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: features must be float32, float16 or bfloat16", op);
  if (f->heads < 1 || f->kv_heads < 1 || f->heads % f->kv_heads != 0 || f->heads > 4096)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: heads must be a positive multiple of the key/value heads (at most 4096)", op);
  if (f->heads / f->kv_heads > 64)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: at most 64 query heads may share a key/value head", op);
  if (f->channels < 1 || f->channels > 128)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: channels must be 1 to 128", op);
  if (f->num_buckets < 0 || f->num_buckets > kMaxBuckets)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: the bias has 1 to %d buckets", op, kMaxBuckets);
  if (!(fabsf(f->scale) <= FLT_MAX)) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: scale must be finite", op);
  if (!pointers) return TBVH_OK;
  if (f->num_buckets > 0 && (!f->bias_table || (!f->bias_edges && f->num_buckets > 1)))
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL bias pointer", op);
  if (!f->keys || !f->values) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL input pointer", op);
  if (!aligned(element_size(f->dtype), f->queries, f->keys, f->values) ||
      (f->num_buckets > 0 && !aligned(4, f->bias_table, f->bias_edges)))
    return misaligned(op);
  return TBVH_OK;
}

// All but the status word, which is the current device's.
AttendArgs common_args(const tbvh_block_geometry* g, const tbvh_attend_features* f, const BlockSetup& s,
                       bool back) {
  AttendArgs a{};
  a.map = s.map;
  a.plan = s.plan;
  a.aabbs = g->node_aabbs;
  a.sorted = g->sorted_indices;
  a.dim = g->dim;
  a.q = f->queries;
  a.k = f->keys;
  a.v = f->values;
  a.heads = f->heads;
  a.kv_heads = f->kv_heads;
  a.channels = f->channels;
  a.group = f->heads / f->kv_heads;
  a.scale = f->scale;
  a.table = f->num_buckets > 0 ? f->bias_table : nullptr;
  a.edges = f->bias_edges;
  a.buckets = f->num_buckets;
  a.splits = 1;
  plan_heads(a, element_size(f->dtype), back);
  return a;
}

struct BackwardSizes {
  size_t delta, most, part, rows, queries;
  size_t total() const { return delta + most + part + rows + queries; }
};

BackwardSizes backward_sizes(const BlockSetup& s, const tbvh_attend_features* f, int splits) {
  BackwardSizes b{};
  b.delta = pad256(size_t(s.total_queries) * f->heads * 4);
  b.most = 256;
  if (f->num_buckets > 0) {
    b.part = pad256(size_t(splits) * s.map.num_tiles * f->heads * f->num_buckets * 4);
    b.rows = pad256(size_t(kTableRows) * f->heads * f->num_buckets * 8);
  }
  if (splits > 1)
    b.queries = size_t(splits) * s.map.num_tiles * f->heads * kTileQueries * padded_channels(f->channels) * 4;
  return b;
}

// Row copies place rows by 32-bit counts of 16-byte words; tensors past 64 GB
// take the narrower copies, which count in 64 bits.
bool words_fit(const BlockSetup& s, const tbvh_attend_features* f) {
  const int64_t size = element_size(f->dtype);
  const int64_t most = std::max(s.total_points * f->kv_heads, s.total_queries * f->heads);
  return most * f->channels * size / 16 < (int64_t(1) << 32);
}

bool pairs_aligned(int channels, const void* p) { return channels % 2 == 0 && uintptr_t(p) % 4 == 0; }

}  // namespace
}  // namespace tbvh

extern "C" {

size_t tbvh_attend_blocks_workspace_size(const tbvh_block_geometry* g, const tbvh_attend_features* f) {
  using namespace tbvh;
  BlockSetup s;
  if (measure_blocks("attend_blocks", g, s) || check_features("attend_blocks", f, false)) return 0;
  const AttendArgs a = common_args(g, f, s, false);
  const int splits = tile_splits(s, a);
  if (splits == 1) return 256;
  return size_t(splits) * s.map.num_tiles * f->heads * kTileQueries * (2 * padded_channels(f->channels) + 2) * 4;
}

int tbvh_attend_blocks(const tbvh_block_geometry* g, const tbvh_attend_features* f, void* out, float* stats,
                       float* out_exact, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tbvh;
  const char* op = "attend_blocks";
  int rc = check_features(op, f, true);
  if (rc) return rc;
  BlockSetup s;
  rc = setup_blocks(op, g, s);
  if (rc) return rc;
  if (s.total_queries == 0) return TBVH_OK;
  if (out_exact && f->dtype == TBVH_F32)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: out_exact is for 16-bit features (out is float32 already)", op);
  if (!f->queries || !out) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL query or output pointer", op);
  if (!aligned(element_size(f->dtype), out) || !aligned(8, stats) || !aligned(4, out_exact, workspace)) return misaligned(op);
  AttendArgs a = common_args(g, f, s, false);
  a.status = device_status_ptr();
  a.splits = tile_splits(s, a);
  const size_t need = tbvh_attend_blocks_workspace_size(g, f);
  if (a.splits > 1 && (workspace == nullptr || workspace_bytes < need))
    return blocks_fail(TBVH_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the required %zu", op,
                       workspace_bytes, need);
  a.width = copy_width(size_t(f->channels) * element_size(f->dtype), f->queries, f->keys, f->values);
  if (!words_fit(s, f)) a.width = std::min(a.width, 8);
  a.wide_out = pairs_aligned(f->channels, out);
  a.out = out;
  a.stats = reinterpret_cast<float2*>(stats);
  a.out_exact = out_exact;
  a.part_row = padded_channels(f->channels) * (out_exact ? 2 : 1) + 2;
  a.part = static_cast<float*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_attend_forward(a, f->dtype, st);
  if (e == cudaSuccess && a.splits > 1) e = launch_attend_merge(a, f->dtype, st);
  return e == cudaSuccess ? TBVH_OK : blocks_cuda_fail(e, op);
}

size_t tbvh_attend_blocks_backward_workspace_size(const tbvh_block_geometry* g, const tbvh_attend_features* f) {
  using namespace tbvh;
  BlockSetup s;
  if (measure_blocks("attend_blocks_backward", g, s) || check_features("attend_blocks_backward", f, false)) return 0;
  return backward_sizes(s, f, tile_splits(s, common_args(g, f, s, true))).total();
}

int tbvh_attend_blocks_backward(const tbvh_block_geometry* g, const tbvh_attend_features* f, const void* out,
                                const float* out_exact, const float* stats, const void* grad_out, void* grad_queries,
                                void* grad_keys, void* grad_values, float* grad_table, void* workspace,
                                size_t workspace_bytes, void* stream) {
  using namespace tbvh;
  const char* op = "attend_blocks_backward";
  int rc = check_features(op, f, true);
  if (rc) return rc;
  BlockSetup s;
  rc = setup_blocks(op, g, s);
  if (rc) return rc;
  if ((grad_keys == nullptr) != (grad_values == nullptr))
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: grad_keys and grad_values must both be given or both be NULL", op);
  if (grad_keys && !g->backward)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: the selection was made without the backward lists", op);
  if (grad_table && f->num_buckets == 0)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: grad_table needs a bias", op);
  if (s.total_queries > 0 && (!f->queries || (!out && !out_exact) || !stats || !grad_out))
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL query, output or gradient pointer", op);
  if (!aligned(element_size(f->dtype), out, grad_out, grad_queries, grad_keys, grad_values) ||
      !aligned(8, stats, workspace) || !aligned(4, out_exact, grad_table))
    return misaligned(op);
  AttendArgs a = common_args(g, f, s, true);
  a.status = device_status_ptr();
  a.splits = tile_splits(s, a);
  const BackwardSizes b = backward_sizes(s, f, a.splits);
  if (workspace == nullptr || workspace_bytes < b.total())
    return blocks_fail(TBVH_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the required %zu", op,
                       workspace_bytes, b.total());
  char* at = static_cast<char*>(workspace);
  a.delta = reinterpret_cast<float*>(at);
  at += b.delta;
  unsigned* most = reinterpret_cast<unsigned*>(at);
  at += b.most;
  float* part = reinterpret_cast<float*>(at);
  at += b.part;
  double* rows = reinterpret_cast<double*>(at);
  at += b.rows;
  a.part = reinterpret_cast<float*>(at);
  a.part_row = padded_channels(f->channels);
  a.stats_in = reinterpret_cast<const float2*>(stats);
  a.grad_out = grad_out;
  a.grad_q = grad_queries;
  a.grad_k = grad_keys;
  a.grad_v = grad_values;
  a.largest = f->dtype == TBVH_F16 && s.total_queries > 0 ? most : nullptr;
  a.table_part = grad_table ? part : nullptr;
  const size_t row_bytes = size_t(f->channels) * element_size(f->dtype);
  a.width = copy_width(row_bytes, f->queries, f->keys, f->values);
  const int grad_width = copy_width(row_bytes, grad_out, nullptr, nullptr);
  if (grad_width < a.width) a.width = grad_width;
  if (!words_fit(s, f)) a.width = std::min(a.width, 8);
  a.wide_out = (!grad_queries || pairs_aligned(f->channels, grad_queries)) &&
               (!grad_keys || (pairs_aligned(f->channels, grad_keys) && pairs_aligned(f->channels, grad_values)));

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  const int values = f->heads * f->num_buckets;
  if (s.total_queries > 0) {
    if (a.largest) e = cudaMemsetAsync(most, 0, 8, st);
    if (a.largest && e == cudaSuccess)
      e = run_largest(static_cast<const __half*>(f->values), s.total_points * f->kv_heads * f->channels, most + 1, st);
    const int64_t pairs = s.total_queries * f->heads;
    if ((pairs + 7) / 8 > INT_MAX) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: too many query rows", op);
    if (e == cudaSuccess) {
      if (f->dtype == TBVH_BF16) e = run_delta<__nv_bfloat16>(grad_out, out, out_exact, a.delta, nullptr, pairs, f->channels, st);
      else if (f->dtype == TBVH_F16) e = run_delta<__half>(grad_out, out, out_exact, a.delta, most, pairs, f->channels, st);
      else e = run_delta<float>(grad_out, out, out_exact, a.delta, nullptr, pairs, f->channels, st);
    }
    if (e == cudaSuccess && (grad_queries || grad_table)) e = launch_attend_grad_q(a, f->dtype, st);
  }
  if (e == cudaSuccess && grad_table) {
    if (s.total_queries == 0) {
      e = cudaMemsetAsync(grad_table, 0, size_t(values) * 4, st);
    } else {
      e = launch_table_sum(part, rows, grad_table, a.splits * s.map.num_tiles, values, st);
    }
  }
  if (e == cudaSuccess && grad_keys) e = launch_attend_grad_kv(a, f->dtype, st);
  return e == cudaSuccess ? TBVH_OK : blocks_cuda_fail(e, op);
}

}  // extern "C"
