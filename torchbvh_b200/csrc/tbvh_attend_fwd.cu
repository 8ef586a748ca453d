// Forward pass of block attention (tbvh_attend_q.cuh) and the joining of its
// splits.
#include "tbvh_attend_q.cuh"
#include "tbvh_kernels.h"

namespace tbvh {

cudaError_t launch_attend_forward(const AttendArgs& a, int dtype, cudaStream_t stream) {
  const cudaError_t e = a.out_exact != nullptr ? launch_attend_forward_exact(a, dtype, stream)
                                               : run_query_tile_by_type<false, false>(a, dtype, stream);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

namespace {

// Joins the splits of one row: with m = max m_s, l = sum l_s 2^(m_s - m) and
// o = sum o_s 2^(m_s - m) / l. One warp a row; a lane has one split's m and l,
// then every 32nd channel of all splits, eight splits in flight.
template <typename T>
__global__ void __launch_bounds__(256) k_merge(AttendArgs a, int cp) {
  const int64_t tile = blockIdx.x;
  const float unit = Units(a.scale).unit;
  const int head = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t stride = a.map.num_tiles * a.heads * kTileQueries * a.part_row;  // floats between splits
  const int rows = a.plan.query_row[tile * kTileQueries + lane];  // a tile's missing queries are its last
  const int there = __popc(__ballot_sync(kFullMask, rows >= 0));
  for (int q = threadIdx.x >> 5; q < there; q += 8) {
    const int row = __shfl_sync(kFullMask, rows, q);
    if (row < 0) continue;
    const float* part = a.part + ((tile * a.heads + head) * kTileQueries + q) * a.part_row;
    const bool mine = lane < a.splits;
    float top = mine ? part[lane * stride] : -INFINITY;
    float sum = mine ? part[lane * stride + 1] : 0.0f;
    float most = top;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(kFullMask, most, d));
    const float base = most == -INFINITY ? 0.0f : most;
    const float w = exp2_fast((top - base) * unit);
    sum *= w;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFullMask, sum, d);
    float o[4] = {}, fine[4] = {};
    const bool exact = a.out_exact != nullptr;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
      const float ws = __shfl_sync(kFullMask, w, s);
      const float* p = part + s * stride + 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (lane + 32 * i < cp) {
          o[i] = fmaf(p[lane + 32 * i], ws, o[i]);
          if (exact) fine[i] = fmaf(p[cp + lane + 32 * i], ws, fine[i]);
        }
      }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / Frag<T>::PEAK_OUT / sum;
    T* out = static_cast<T*>(a.out) + (int64_t(row) * a.heads + head) * a.channels;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (lane + 32 * i < a.channels) {
        out[lane + 32 * i] = Frag<T>::from_float(o[i] * inv);
        if (exact) a.out_exact[(int64_t(row) * a.heads + head) * a.channels + lane + 32 * i] = (o[i] + fine[i]) * inv;
      }
    }
    if (a.stats != nullptr && lane == 0) a.stats[int64_t(row) * a.heads + head] = row_stats(most, sum);
  }
}

}  // namespace

cudaError_t launch_attend_merge(const AttendArgs& a, int dtype, cudaStream_t stream) {
  const dim3 grid(unsigned(a.map.num_tiles), unsigned(a.heads));
  const int cp = padded_channels(a.channels);
  if (dtype == TBVH_BF16) k_merge<__nv_bfloat16><<<grid, 256, 0, stream>>>(a, cp);
  else if (dtype == TBVH_F16) k_merge<__half><<<grid, 256, 0, stream>>>(a, cp);
  else k_merge<float><<<grid, 256, 0, stream>>>(a, cp);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace tbvh
