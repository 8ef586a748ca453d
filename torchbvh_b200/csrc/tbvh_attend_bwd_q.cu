// Backward pass of block attention, sums over keys (tbvh_attend_q.cuh), and the
// joining of its splits.
#include "tbvh_attend_q.cuh"
#include "tbvh_kernels.h"

namespace tbvh {
namespace {

// dQ of a tile and head: the sum of its splits, in their order, times the scale.
// One warp a row; a lane has every 32nd channel.
template <typename T>
__global__ void __launch_bounds__(256) k_join_grad(AttendArgs a) {
  const int64_t tile = blockIdx.x;
  const int head = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t stride = a.map.num_tiles * a.heads * kTileQueries * a.part_row;  // floats between splits
  const float back = a.scale / gradient_lift<T>(a);
  for (int q = threadIdx.x >> 5; q < kTileQueries; q += 8) {
    const int row = a.plan.query_row[tile * kTileQueries + q];
    if (row < 0) continue;
    const float* part = a.part + ((tile * a.heads + head) * kTileQueries + q) * a.part_row;
    T* out = static_cast<T*>(a.grad_q) + (int64_t(row) * a.heads + head) * a.channels;
    for (int i = lane; i < a.channels; i += 32) {
      float sum = 0.0f;
#pragma unroll 8
      for (int s = 0; s < a.splits; ++s) sum += part[s * stride + i];
      out[i] = Frag<T>::from_float(sum * back);
    }
  }
}

}  // namespace

cudaError_t launch_attend_grad_q(const AttendArgs& a, int dtype, cudaStream_t stream) {
  const cudaError_t e = run_query_tile_by_type<true, false>(a, dtype, stream);
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (a.splits == 1 || a.grad_q == nullptr) return cudaSuccess;
  const dim3 grid(unsigned(a.map.num_tiles), unsigned(a.heads));
  if (dtype == TBVH_BF16) k_join_grad<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else if (dtype == TBVH_F16) k_join_grad<__half><<<grid, 256, 0, stream>>>(a);
  else k_join_grad<float><<<grid, 256, 0, stream>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace tbvh
