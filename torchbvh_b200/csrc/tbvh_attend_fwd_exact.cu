// Forward pass of block attention that also keeps its float32 output
// (tbvh_attend_q.cuh).
#include "tbvh_attend_q.cuh"

namespace tbvh {

cudaError_t launch_attend_forward_exact(const AttendArgs& a, int dtype, cudaStream_t stream) {
  return run_query_tile_by_type<false, true>(a, dtype, stream);
}

}  // namespace tbvh
