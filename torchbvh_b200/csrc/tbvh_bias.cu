// Learned bias of neighbour lists by distance bucket, and the gradient of its
// table (also the last step of block attention's table gradient).
//
// Forward: 4 bytes read and 4 written a value, a bucket lookup and a table read
// in shared memory. Backward: 8 bytes read a value; every thread sums into a
// column of its own of a [bucket][thread] array in shared memory (bank = lane,
// no conflicts, no atomics, a fixed order), columns and thread blocks are then
// joined in a fixed order.
#include <climits>

#include "tbvh_attend.cuh"
#include "tbvh_kernels.h"

namespace tbvh {
namespace {

// out[y][i] = sum of part rows.
// Block (x, y) sums rows y * 8 + w, + 8 gridDim.y, ... of 32 values with 8 warps, in
// 64 bits and a fixed order; a second launch sums the gridDim.y results.
template <typename In, typename Out>
__global__ void __launch_bounds__(256) k_table_sum(const In* part, Out* out, int64_t rows, int values) {
  __shared__ double s_sum[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  double sum = 0.0;
  if (i < values)
    for (int64_t t = int64_t(blockIdx.y) * 8 + warp; t < rows; t += int64_t(gridDim.y) * 8)
      sum += double(part[t * values + i]);
  s_sum[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && i < values) {
    for (int w = 1; w < 8; ++w) sum += s_sum[w][lane];
    out[int64_t(blockIdx.y) * values + i] = Out(sum);
  }
}

constexpr int kBiasThreads = 256;    // backward
constexpr int kForwardThreads = 512;
constexpr int kBiasTable = 8192;  // table values kept in shared memory

struct BiasArgs {
  const float* d2;
  const float* table;
  const float* edges;
  const float* grad;
  float* out;   // forward: bias; backward: partial tables [gridDim.x][heads][buckets]
  int64_t rows, k;
  int heads, buckets;
  bool per_head;
};

// W values of a row at once (W = 4: k a multiple of 4 and 16-byte addresses).
// Few, large thread blocks: each makes the bucket table once.
template <int W>
__global__ void __launch_bounds__(kForwardThreads) k_bias(BiasArgs a, bool table_here) {
  __shared__ BucketTable s_buckets;
  extern __shared__ float s_table[];
  const int values = a.heads * a.buckets;
  if (table_here)
    for (int i = threadIdx.x; i < values; i += kForwardThreads) s_table[i] = a.table[i];
  s_buckets.make(a.edges, a.buckets - 1);
  __syncthreads();
  const float* table = table_here ? s_table : a.table;
  const int64_t per_row = a.k / W;
  const int64_t lists = a.per_head ? a.rows * a.heads : a.rows;
  const int64_t total = lists * per_row, step = int64_t(gridDim.x) * kForwardThreads;
  const bool small = total <= UINT_MAX;
  auto read = [&](int64_t i, float (&d)[W]) {
    if constexpr (W == 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(a.d2) + i);
      d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
    } else {
      d[0] = __ldg(a.d2 + i);
    }
  };
  int64_t i = int64_t(blockIdx.x) * kForwardThreads + threadIdx.x;
  float d[W], next[W];
  if (i < total) read(i, d);
  for (; i < total; i += step) {
    if (i + step < total) read(i + step, next);
    const int64_t list = small ? int64_t(uint32_t(i) / uint32_t(per_row)) : i / per_row;
    const int64_t at = (i - list * per_row) * W;
    uint32_t b[W];
#pragma unroll
    for (int w = 0; w < W; ++w) b[w] = s_buckets.find_any(d[w]);
    auto store = [&](int64_t row_head, int head) {
      const float* t = table + head * a.buckets;
      float* o = a.out + row_head * a.k + at;
      if constexpr (W == 4) *reinterpret_cast<float4*>(o) = make_float4(t[b[0]], t[b[1]], t[b[2]], t[b[3]]);
      else *o = t[b[0]];
    };
    if (a.per_head) store(list, int(small ? uint32_t(list) % uint32_t(a.heads) : list % a.heads));
    else
      for (int h = 0; h < a.heads; ++h) store(list * a.heads + h, h);
#pragma unroll
    for (int w = 0; w < W; ++w) d[w] = next[w];
  }
}

// blockIdx.y: head. Thread blocks of a head stride over its rows; the next
// iteration's values are in flight while this one's are summed.
template <int W>
__global__ void __launch_bounds__(kBiasThreads) k_bias_grad(BiasArgs a) {
  __shared__ BucketTable s_buckets;
  extern __shared__ float s_hist[];  // [buckets][threads]
  const int tid = threadIdx.x, lane = tid & 31, head = blockIdx.y;
  const int64_t per_row = a.k / W;
  const int64_t total = a.rows * per_row, step = int64_t(gridDim.x) * kBiasThreads;
  const bool small = total <= UINT_MAX;
  auto read = [&](int64_t i, float (&d)[W], float (&x)[W]) {
    const int64_t row = small ? int64_t(uint32_t(i) / uint32_t(per_row)) : i / per_row;
    const int64_t at = (i - row * per_row) * W;
    const float* p = a.d2 + (a.per_head ? row * a.heads + head : row) * a.k + at;
    const float* q = a.grad + (row * a.heads + head) * a.k + at;
    if constexpr (W == 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p)), u = __ldg(reinterpret_cast<const float4*>(q));
      d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
      x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    } else {
      d[0] = __ldg(p);
      x[0] = __ldg(q);
    }
  };
  int64_t i = int64_t(blockIdx.x) * kBiasThreads + tid;
  float d[W], x[W], next_d[W], next_x[W];
  if (i < total) read(i, d, x);
  for (int b = 0; b < a.buckets; ++b) s_hist[b * kBiasThreads + tid] = 0.0f;
  s_buckets.make(a.edges, a.buckets - 1);
  __syncthreads();
  for (; i < total; i += step) {
    if (i + step < total) read(i + step, next_d, next_x);
#pragma unroll
    for (int w = 0; w < W; ++w) s_hist[s_buckets.find_any(d[w]) * kBiasThreads + tid] += x[w];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      d[w] = next_d[w];
      x[w] = next_x[w];
    }
  }
  for (int b = 0; b < a.buckets; ++b) {
    float v = s_hist[b * kBiasThreads + tid];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFullMask, v, d);
    if (lane == 0) s_hist[b * kBiasThreads + tid] = v;
  }
  __syncthreads();
  for (int b = tid; b < a.buckets; b += kBiasThreads) {
    float v = 0.0f;
    for (int w = 0; w < kBiasThreads / 32; ++w) v += s_hist[b * kBiasThreads + w * 32];
    a.out[(int64_t(blockIdx.x) * a.heads + head) * a.buckets + b] = v;
  }
}

bool by_four(int64_t k, const void* a, const void* b) {
  return k % 4 == 0 && (uintptr_t(a) | uintptr_t(b)) % 16 == 0;
}

// Thread blocks of one head of the backward pass: about four an SM in all, at
// least eight values a thread.
int64_t grad_blocks(int64_t rows, int heads, int64_t k) {
  int64_t want = (4 * 148 + heads - 1) / heads;
  const int64_t most = (rows * k + 8 * kBiasThreads - 1) / (8 * kBiasThreads);
  if (want > most) want = most;
  return want < 1 ? 1 : want;
}

size_t pad256(size_t v) { return (v + 255) / 256 * 256; }

int check_bias(const char* op, int64_t rows, int heads, int64_t k, int buckets) {
  if (rows < 0 || k < 0 || rows > INT64_MAX / 8192 || k > INT_MAX)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: bad number of rows or values", op);
  if (heads < 1 || heads > 4096) return blocks_fail(TBVH_ERR_BAD_ARG, "%s: heads must be 1 to 4096", op);
  if (buckets < 1 || buckets > kMaxBuckets)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: the bias has 1 to %d buckets", op, kMaxBuckets);
  return TBVH_OK;
}

int use_device(const char* op, int device) {
  int cur = -1;
  if (device < 0 || (cudaGetDevice(&cur) == cudaSuccess && cur == device)) return TBVH_OK;
  const cudaError_t e = cudaSetDevice(device);
  return e == cudaSuccess ? TBVH_OK : blocks_cuda_fail(e, op);
}

}  // namespace

cudaError_t launch_table_sum(const float* part, double* scratch, float* grad_table, int64_t rows, int values,
                             cudaStream_t stream) {
  const unsigned columns = unsigned((values + 31) / 32);
  if (rows <= 256) {  // 32 rows a warp: one launch is sooner done than two
    k_table_sum<float, float><<<dim3(columns, 1), 256, 0, stream>>>(part, grad_table, rows, values);
    count_launches(1);
    return cudaGetLastError();
  }
  const int rows_out = rows < 8 * kTableRows ? int((rows + 7) / 8) : kTableRows;
  k_table_sum<float, double><<<dim3(columns, unsigned(rows_out)), 256, 0, stream>>>(part, scratch, rows, values);
  k_table_sum<double, float><<<dim3(columns, 1), 256, 0, stream>>>(scratch, grad_table, rows_out, values);
  count_launches(2);
  return cudaGetLastError();
}

}  // namespace tbvh

extern "C" {

int tbvh_distance_bias(int device, const float* squared_distances, int64_t rows, int heads, int64_t k, int per_head,
                       const float* table, const float* edges, int num_buckets, float* out, void* stream) {
  using namespace tbvh;
  const char* op = "distance_bias";
  int rc = check_bias(op, rows, heads, k, num_buckets);
  if (rc) return rc;
  if (rows == 0 || k == 0) return TBVH_OK;
  if (!squared_distances || !table || (!edges && num_buckets > 1) || !out)
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL pointer", op);
  rc = use_device(op, device);
  if (rc) return rc;
  BiasArgs a{squared_distances, table, edges, nullptr, out, rows, k, heads, num_buckets, per_head != 0};
  const bool four = by_four(k, squared_distances, out);
  const int64_t items = rows * (per_head ? heads : 1) * (four ? k / 4 : k);
  int64_t grid = (items + kForwardThreads - 1) / kForwardThreads;
  if (grid > 4 * 148) grid = 4 * 148;
  const bool here = heads * num_buckets <= kBiasTable;
  const size_t smem = here ? size_t(heads) * num_buckets * 4 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (four) k_bias<4><<<unsigned(grid), kForwardThreads, smem, st>>>(a, here);
  else k_bias<1><<<unsigned(grid), kForwardThreads, smem, st>>>(a, here);
  count_launches(1);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TBVH_OK : blocks_cuda_fail(e, op);
}

size_t tbvh_distance_bias_backward_workspace_size(int64_t rows, int heads, int64_t k, int num_buckets) {
  using namespace tbvh;
  if (check_bias("distance_bias_backward", rows, heads, k, num_buckets)) return 0;
  return pad256(size_t(grad_blocks(rows, heads, k)) * heads * num_buckets * 4) +
         size_t(kTableRows) * heads * num_buckets * 8;
}

int tbvh_distance_bias_backward(int device, const float* squared_distances, int64_t rows, int heads, int64_t k,
                                int per_head, const float* edges, int num_buckets, const float* grad_out,
                                float* grad_table, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tbvh;
  const char* op = "distance_bias_backward";
  int rc = check_bias(op, rows, heads, k, num_buckets);
  if (rc) return rc;
  const bool none = rows == 0 || k == 0;
  if (!grad_table || (!none && (!squared_distances || (!edges && num_buckets > 1) || !grad_out)))
    return blocks_fail(TBVH_ERR_BAD_ARG, "%s: NULL pointer", op);
  const size_t need = tbvh_distance_bias_backward_workspace_size(rows, heads, k, num_buckets);
  if (workspace == nullptr || workspace_bytes < need)
    return blocks_fail(TBVH_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the required %zu", op,
                       workspace_bytes, need);
  rc = use_device(op, device);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (none) {
    e = cudaMemsetAsync(grad_table, 0, size_t(heads) * num_buckets * 4, st);
    return e == cudaSuccess ? TBVH_OK : blocks_cuda_fail(e, op);
  }
  const int64_t blocks = grad_blocks(rows, heads, k);
  float* part = static_cast<float*>(workspace);
  double* scratch = reinterpret_cast<double*>(static_cast<char*>(workspace) +
                                              pad256(size_t(blocks) * heads * num_buckets * 4));
  BiasArgs a{squared_distances, nullptr, edges, grad_out, part, rows, k, heads, num_buckets, per_head != 0};
  const size_t smem = size_t(num_buckets) * kBiasThreads * 4;
  const bool four = by_four(k, squared_distances, grad_out);
  static_assert(sizeof(BucketTable) + 4 * kMaxBuckets <= kStaticSmem, "static arrays of k_bias_grad");
  e = four ? allow_smem(k_bias_grad<4>, smem) : allow_smem(k_bias_grad<1>, smem);
  if (e != cudaSuccess) return blocks_cuda_fail(e, op);
  const dim3 grid{unsigned(blocks), unsigned(heads)};
  if (four) k_bias_grad<4><<<grid, kBiasThreads, smem, st>>>(a);
  else k_bias_grad<1><<<grid, kBiasThreads, smem, st>>>(a);
  count_launches(1);
  e = cudaGetLastError();
  if (e == cudaSuccess) e = launch_table_sum(part, scratch, grad_table, blocks, heads * num_buckets, st);
  return e == cudaSuccess ? TBVH_OK : blocks_cuda_fail(e, op);
}

}  // extern "C"
