// Backward pass of block attention, sums over keys (tbvh_attend_q.cuh).
#include "tbvh_attend_q.cuh"
#include "tbvh_kernels.h"

namespace tbvh {

cudaError_t launch_attend_grad_q(const AttendArgs& a, int dtype, cudaStream_t stream) {
  const cudaError_t e = run_query_tile_by_type<true, false>(a, dtype, stream);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace tbvh
