// Backward pass of block attention, sums over queries (tbvh_attend_kv.cuh).
#include "tbvh_attend_kv.cuh"
#include "tbvh_kernels.h"

namespace tbvh {

cudaError_t launch_attend_grad_kv(const AttendArgs& a, int dtype, cudaStream_t stream) {
  const cudaError_t e = dtype == TBVH_BF16  ? run_key_block_by_channels<__nv_bfloat16>(a, stream)
                        : dtype == TBVH_F16 ? run_key_block_by_channels<__half>(a, stream)
                                            : run_key_block_by_channels<float>(a, stream);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace tbvh
