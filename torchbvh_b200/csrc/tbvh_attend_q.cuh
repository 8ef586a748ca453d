// Block attention by query tile: the forward pass, and the part of the backward
// pass that sums over keys (gradients of the queries and of the bias table).
//
// A thread block serves one tile (32 queries, neighbours in space) and up to
// four query heads; a warp has one head and 16 of the queries. The block walks
// the tile's entries (64 leaves each, union of what its queries selected) in
// steps of 32 leaves: key and value rows come by asynchronous copies straight
// from the caller's order (sorted_indices), two stages deep, while the previous
// step is computed. A warp none of whose queries selected the entry skips it.
// Distance buckets are the same for every head: the block computes them once a
// step, one byte a pair; a score reads a byte and the head's bias from shared
// memory, and the bias starts the accumulator of its product.
//
//   forward    m, l: running maximum and sum (32 bits); o: sum of p V
//              o <- o 2^(m_old - m) + p V in one pass over the keys
//   backward   p = 2^(z - lse), dS = p (dO V^T - <dO, O>)
//              dQ = scale sum dS K;  dT[h][bucket] += dS
//
// EXACT (forward, 16-bit features whose bias table trains): the parts of the
// probabilities that 16 bits do not hold go through a second product of their
// own, kept apart, so that the output's bits do not depend on it; both sums
// together are the float32 output that <dO, O> is taken from.
//
// A row that did not select the entry keeps its sums by selection, not by
// masking its scores: what it computes there is dropped, so non-finite keys and
// values reach only the rows that attend to them.
#pragma once

#include "tbvh_attend.cuh"

namespace tbvh {

constexpr int kStepLeaves = 32;

struct QueryTileSmem {
  uint32_t k, v, q, d, bias, buckets, pts, rows, qrows, table, hist, total;
};

__host__ __device__ inline QueryTileSmem query_tile_smem(int size, int cp, int kvs, int heads, bool back, bool bias,
                                                         int buckets) {
  QueryTileSmem s{};
  const uint32_t ld = uint32_t(cp + 16 / size);
  uint32_t at = 0;
  auto take = [&](uint32_t bytes) {
    const uint32_t was = at;
    at += (bytes + 15) / 16 * 16;
    return was;
  };
  s.k = take(2 * kvs * kStepLeaves * ld * size);
  s.v = take(2 * kvs * kStepLeaves * ld * size);
  s.q = take(heads * kTileQueries * ld * size);
  s.d = back ? take(heads * kTileQueries * ld * size) : 0;
  s.rows = take(2 * kStepLeaves * 4);
  s.qrows = take(kTileQueries * 4);
  if (bias) {
    s.bias = take(heads * kMaxBuckets * 4);
    s.buckets = take(2 * kTileQueries * (kStepLeaves + 4));
    s.pts = take(2 * 3 * kStepLeaves * 4);
    s.table = take(sizeof(BucketTable));
    if (back) s.hist = take(uint32_t(buckets) * heads * 64 * 4);
  }
  s.total = at;
  return s;
}

// Registers: with 32 padded channels three blocks of eight warps share an SM.
template <typename T, int CP, bool BACK, bool EXACT>
__global__ void __launch_bounds__(256, CP <= 32 ? (BACK || EXACT || sizeof(T) == 4 ? 2 : 3) : CP <= 64 ? 2 : 1)
    k_query_tile(AttendArgs a) {
  using F = Frag<T>;
  constexpr int LD = Tile<T, CP>::LD;
  constexpr int NT = kStepLeaves / 8;
  constexpr int STEPS = kStepLeaves / F::STEP;
  constexpr bool HELD = sizeof(T) == 2 ? CP <= 64 : CP <= 32 && !BACK;
  constexpr int HOLD = HELD ? CP / F::STEP : 1;
  constexpr int BROW = kStepLeaves + 4;  // bytes of one query's bucket row
  extern __shared__ __align__(16) char smem[];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t tile = blockIdx.x;
  const HeadSpan span(a, blockIdx.y);
  const BlockCloud c = a.map.of_tile(tile);
  const bool bias = a.table != nullptr;
  const QueryTileSmem off = query_tile_smem(sizeof(T), CP, a.kv_cta, a.heads_cta, BACK, bias, a.buckets);
  T* s_k = reinterpret_cast<T*>(smem + off.k);
  T* s_v = reinterpret_cast<T*>(smem + off.v);
  T* s_q = reinterpret_cast<T*>(smem + off.q);
  T* s_d = reinterpret_cast<T*>(smem + off.d);
  int* s_rows = reinterpret_cast<int*>(smem + off.rows);
  int* s_qrows = reinterpret_cast<int*>(smem + off.qrows);
  float* s_bias = reinterpret_cast<float*>(smem + off.bias);
  uint8_t* s_buckets = reinterpret_cast<uint8_t*>(smem + off.buckets);
  float* s_pts = reinterpret_cast<float*>(smem + off.pts);
  BucketTable& s_table = *reinterpret_cast<BucketTable*>(smem + off.table);
  float* s_hist = reinterpret_cast<float*>(smem + off.hist);
  const int kv_tile = kStepLeaves * LD, q_tile = kTileQueries * LD;
  const int stage = a.kv_cta * kv_tile;

  const int all = a.plan.tile_count[tile];
  const int splits = BACK ? 1 : a.splits;
  const int from = int(int64_t(all) * blockIdx.z / splits), count = int(int64_t(all) * (blockIdx.z + 1) / splits) - from;
  const int steps = 2 * count;
  const uint2* entries = a.plan.entries + tile * a.plan.capacity + from;
  const int64_t leaves = bias ? leaf_row0(c) : 0;
  // Logits are kept as z / unit: the bias enters the products' accumulators
  // divided by the scale, and scale and base change are one factor in the
  // exponential. Scales that this does not suit (negative, tiny, huge) are
  // applied to the products instead.
  const bool folded = a.scale >= 0x1p-30f && a.scale <= 0x1p30f;
  const float unit = folded ? a.scale * kLog2e : 1.0f;
  const float bias_unit = folded ? 1.0f / a.scale : kLog2e;

  if (tid < kTileQueries) s_qrows[tid] = a.plan.query_row[tile * kTileQueries + tid];
  // Rows (and points) of step `i`, one leaf a lane of the first warp.
  int next_row = -1;
  float next_pt[3] = {0.0f, 0.0f, 0.0f};
  auto fetch = [&](int i) {
    if (tid < kStepLeaves && i < steps) {
      const int64_t leaf = int64_t(entries[i >> 1].x) * kBlockLeaves + (i & 1) * kStepLeaves + tid;
      next_row = key_row(a, c, leaf);
      if (bias) {
        const float* p = a.aabbs + (leaves + leaf) * 2 * a.dim;
        for (int x = 0; x < 3; ++x) next_pt[x] = leaf < c.n && x < a.dim ? p[x] : 0.0f;
      }
    }
  };
  auto put = [&](int i) {
    if (tid < kStepLeaves && i < steps) {
      const int slot = i & 1;
      s_rows[slot * kStepLeaves + tid] = next_row;
      if (bias)
        for (int x = 0; x < 3; ++x) s_pts[(slot * 3 + x) * kStepLeaves + tid] = next_pt[x];
    }
  };
  auto copy = [&](int i) {
    if (i < steps) {
      const int slot = i & 1;
      const int* rows = s_rows + slot * kStepLeaves;
      copy_rows<T, CP>(s_k + slot * stage, kv_tile, static_cast<const T*>(a.k), rows, kStepLeaves, a.kv_heads,
                       a.channels, span.kv0, span.kvs, a.width);
      copy_rows<T, CP>(s_v + slot * stage, kv_tile, static_cast<const T*>(a.v), rows, kStepLeaves, a.kv_heads,
                       a.channels, span.kv0, span.kvs, a.width);
    }
    cp_commit();
  };
  // Distance buckets of step i, times four (byte offsets into a bias row): a
  // thread has one query (the same in every step where the block has 256
  // threads) and four neighbouring leaves.
  auto sort_pairs = [&](int i) {
    if (bias && i < steps) {
      const int slot = i & 1;
      for (int u = tid; u < kTileQueries * kStepLeaves / 4; u += blockDim.x) {
        const int q = u / (kStepLeaves / 4), k4 = u % (kStepLeaves / 4) * 4;
        const float* qp = a.plan.query_point + tile * 3 * kTileQueries + q;
        const float qx = __ldg(qp), qy = __ldg(qp + kTileQueries), qz = __ldg(qp + 2 * kTileQueries);
        const float* p = s_pts + slot * 3 * kStepLeaves + k4;
        const float4 px = *reinterpret_cast<const float4*>(p);
        const float4 py = *reinterpret_cast<const float4*>(p + kStepLeaves);
        const float4 pz = *reinterpret_cast<const float4*>(p + 2 * kStepLeaves);
        const bool three = a.dim == 3;
        const uint32_t b0 = s_table.find(pair_distance(qx, qy, qz, px.x, py.x, pz.x, three));
        const uint32_t b1 = s_table.find(pair_distance(qx, qy, qz, px.y, py.y, pz.y, three));
        const uint32_t b2 = s_table.find(pair_distance(qx, qy, qz, px.z, py.z, pz.z, three));
        const uint32_t b3 = s_table.find(pair_distance(qx, qy, qz, px.w, py.w, pz.w, three));
        *reinterpret_cast<uint32_t*>(s_buckets + (slot * kTileQueries + q) * BROW + k4) =
            (b0 | b1 << 8 | b2 << 16 | b3 << 24) << 2;
      }
    }
  };

  clear_padding<T, CP>(s_k, 2 * a.kv_cta * kStepLeaves, a.channels);
  clear_padding<T, CP>(s_v, 2 * a.kv_cta * kStepLeaves, a.channels);
  clear_padding<T, CP>(s_q, a.heads_cta * kTileQueries, a.channels);
  if constexpr (BACK) clear_padding<T, CP>(s_d, a.heads_cta * kTileQueries, a.channels);
  fetch(0);
  put(0);
  if (bias) {
    for (int i = tid; i < span.heads * a.buckets; i += blockDim.x)
      s_bias[(i / a.buckets) * kMaxBuckets + i % a.buckets] = a.table[int64_t(span.h0) * a.buckets + i] * bias_unit;
    if constexpr (BACK)
      for (int i = tid; i < a.buckets * int(blockDim.x); i += blockDim.x) s_hist[i] = 0.0f;
  }
  __syncthreads();
  copy_rows<T, CP>(s_q, q_tile, static_cast<const T*>(a.q), s_qrows, kTileQueries, a.heads, a.channels, span.h0,
                   span.heads, a.width);
  if constexpr (BACK)
    copy_rows<T, CP>(s_d, q_tile, static_cast<const T*>(a.grad_out), s_qrows, kTileQueries, a.heads, a.channels,
                     span.h0, span.heads, a.width);
  copy(0);
  fetch(1);
  put(1);
  if (bias) {
    s_table.make(a.edges, a.buckets - 1);
    __syncthreads();
  }
  sort_pairs(0);
  cp_wait<0>();
  __syncthreads();

  const int head = warp >> 1, half = warp & 1;
  const bool mine = head < span.heads;
  const int kv = mine ? (span.h0 + head) / a.group - span.kv0 : 0;
  const int g = lane >> 2, t = lane & 3;
  const T* q_rows = s_q + head * q_tile;
  const T* d_rows = s_d + head * q_tile;
  const char* head_bias = reinterpret_cast<const char*>(s_bias + head * kMaxBuckets);
  char* hist = reinterpret_cast<char*>(s_hist + tid);

  typename F::A held_q[HOLD], held_d[BACK ? HOLD : 1];
  if constexpr (HELD) {
    if (mine) hold<T, CP>(held_q, q_rows, half * 16, lane);
    if constexpr (BACK)
      if (mine) hold<T, CP>(held_d, d_rows, half * 16, lane);
  }
  float acc[CP / 8][4] = {};
  float fine[EXACT ? CP / 8 : 1][4] = {};
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};  // forward: running maximum, sum
  float lse[2] = {INFINITY, INFINITY}, delta[2] = {0.0f, 0.0f};  // backward
  float lift = 1.0f;  // float16: power of two that brings the gradients to order 1
  if constexpr (BACK) {
    lift = gradient_lift<T>(a);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = s_qrows[half * 16 + g + 8 * r];
      if (mine && row >= 0) {
        lse[r] = a.lse_in[int64_t(row) * a.heads + span.h0 + head];
        delta[r] = a.delta[int64_t(row) * a.heads + span.h0 + head] * lift;
      }
    }
  }

  for (int i = 0; i < steps; ++i) {
    cp_wait<0>();
    __syncthreads();
    copy(i + 1);
    fetch(i + 2);
    sort_pairs(i + 1);
    const uint2 entry = entries[i >> 1];
    const unsigned mask = entry.y >> (half * 16);
    const int64_t left = c.n - int64_t(entry.x) * kBlockLeaves - (i & 1) * kStepLeaves;
    if (mine && (mask & 0xffffu) && left > 0) {
      const int slot = i & 1;
      const T* k_tile = s_k + slot * stage + kv * kv_tile;
      const T* v_tile = s_v + slot * stage + kv * kv_tile;
      const bool on[2] = {(mask >> g & 1u) != 0, (mask >> (g + 8) & 1u) != 0};
      const uint8_t* near = s_buckets + (slot * kTileQueries + half * 16 + g) * BROW + 2 * t;
      float s[NT][4];
      auto read_bias = [&]() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint32_t lo = *reinterpret_cast<const uint16_t*>(near + n * 8);
          const uint32_t hi = *reinterpret_cast<const uint16_t*>(near + 8 * BROW + n * 8);
          s[n][0] = *reinterpret_cast<const float*>(head_bias + (lo & 255));
          s[n][1] = *reinterpret_cast<const float*>(head_bias + (lo >> 8));
          s[n][2] = *reinterpret_cast<const float*>(head_bias + (hi & 255));
          s[n][3] = *reinterpret_cast<const float*>(head_bias + (hi >> 8));
        }
      };
      if (bias && folded) {
        read_bias();
        multiply_nk<T, CP, NT, HELD>(s, held_q, q_rows, half * 16, k_tile, 0, lane);
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
        multiply_nk<T, CP, NT, HELD>(s, held_q, q_rows, half * 16, k_tile, 0, lane);
        if (!folded) {
          float x[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[n][j] = s[n][j] * (a.scale * kLog2e);
              s[n][j] = 0.0f;
            }
          if (bias) read_bias();
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] += x[n][j];
        }
      }
      if (left < kStepLeaves) {  // the cloud's last leaves
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n * 8 + 2 * t + (j & 1) >= left) s[n][j] = -INFINITY;
      }
      if constexpr (!BACK) {
        float shrink[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float most = top[r];
#pragma unroll
          for (int n = 0; n < NT; ++n) most = fmaxf(most, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
          most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
          most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
          const float base = most == -INFINITY ? 0.0f : most * unit;  // nothing yet: all p are 0
          shrink[r] = exp2_fast(fmaf(top[r], unit, -base));
          float add = 0.0f;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              s[n][2 * r + j] = exp2_fast(fmaf(s[n][2 * r + j], unit, -base));
              add += s[n][2 * r + j];
            }
          }
          if (on[r]) {
            top[r] = most;
            sum[r] = fmaf(sum[r], shrink[r], add);
          }
        }
#pragma unroll
        for (int n0 = 0; n0 < CP / 8; n0 += kChannelGroup) {
          float part[kChannelGroup][4] = {}, low[EXACT ? kChannelGroup : 1][4] = {};
#pragma unroll
          for (int st = 0; st < STEPS; ++st) {
            typename F::A p, rest;
            from_acc<T>(p, s, st);
            if constexpr (EXACT) rest_of_acc<T>(rest, p, s, st);
#pragma unroll
            for (int j = 0; j < kChannelGroup / 2; ++j) {
              typename F::B b;
              F::pair_kn(b, v_tile, LD, st * F::STEP, (n0 + 2 * j) * 8, lane);
              F::mma(part[2 * j], p, b[0], b[1]);
              F::mma(part[2 * j + 1], p, b[2], b[3]);
              if constexpr (EXACT) {
                F::mma(low[2 * j], rest, b[0], b[1]);
                F::mma(low[2 * j + 1], rest, b[2], b[3]);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < kChannelGroup; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (on[x >> 1]) {
                acc[n0 + j][x] = fmaf(acc[n0 + j][x], shrink[x >> 1], part[j][x]);
                if constexpr (EXACT) fine[n0 + j][x] = fmaf(fine[n0 + j][x], shrink[x >> 1], low[j][x]);
              }
        }
      } else {
        float ds[NT][4] = {};
        multiply_nk<T, CP, NT, HELD>(ds, held_d, d_rows, half * 16, v_tile, 0, lane);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            ds[n][j] = exp2_fast(fmaf(s[n][j], unit, -lse[j >> 1])) * fmaf(ds[n][j], lift, -delta[j >> 1]);
        if (bias) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (on[r]) {
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint32_t b = *reinterpret_cast<const uint16_t*>(near + r * 8 * BROW + n * 8);
                // Each thread has a column of its own.
                *reinterpret_cast<float*>(hist + (b & 255) * blockDim.x) += ds[n][2 * r];
                *reinterpret_cast<float*>(hist + (b >> 8) * blockDim.x) += ds[n][2 * r + 1];
              }
            }
          }
        }
#pragma unroll
        for (int n0 = 0; n0 < CP / 8; n0 += kChannelGroup) {
          float part[kChannelGroup][4] = {};
#pragma unroll
          for (int st = 0; st < STEPS; ++st) {
            typename F::A p;
            from_acc<T>(p, ds, st);
#pragma unroll
            for (int j = 0; j < kChannelGroup / 2; ++j) {
              typename F::B b;
              F::pair_kn(b, k_tile, LD, st * F::STEP, (n0 + 2 * j) * 8, lane);
              F::mma(part[2 * j], p, b[0], b[1]);
              F::mma(part[2 * j + 1], p, b[2], b[3]);
            }
          }
#pragma unroll
          for (int j = 0; j < kChannelGroup; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (on[x >> 1]) acc[n0 + j][x] += part[j][x];
        }
      }
    }
    put(i + 2);
  }

  if (mine) {
    if constexpr (!BACK) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        sum[r] += __shfl_xor_sync(kFullMask, sum[r], 1);
        sum[r] += __shfl_xor_sync(kFullMask, sum[r], 2);
        const int q = half * 16 + g + 8 * r;
        const int row = s_qrows[q];
        if (splits > 1) {
          const int64_t slot = ((int64_t(blockIdx.z) * a.map.num_tiles + tile) * a.heads + span.h0 + head) *
                                   kTileQueries + q;
          float* part = a.part + slot * a.part_row;
          if (t == 0) {
            part[0] = top[r] * unit;
            part[1] = sum[r];
          }
#pragma unroll
          for (int n = 0; n < CP / 8; ++n) {
            part[2 + n * 8 + 2 * t] = acc[n][2 * r];
            part[2 + n * 8 + 2 * t + 1] = acc[n][2 * r + 1];
            if constexpr (EXACT) {
              part[2 + CP + n * 8 + 2 * t] = fine[n][2 * r];
              part[2 + CP + n * 8 + 2 * t + 1] = fine[n][2 * r + 1];
            }
          }
          continue;
        }
        if (row < 0) continue;
        const float inv = sum[r] == 0.0f ? 0.0f : 1.0f / sum[r];
        T* out = static_cast<T*>(a.out) + (int64_t(row) * a.heads + span.h0 + head) * a.channels;
#pragma unroll
        for (int n = 0; n < CP / 8; ++n)
          store_pair(out, n * 8 + 2 * t, a.channels, acc[n][2 * r] * inv, acc[n][2 * r + 1] * inv, a.wide_out);
        if constexpr (EXACT) {
          float* exact = a.out_exact + (int64_t(row) * a.heads + span.h0 + head) * a.channels;
#pragma unroll
          for (int n = 0; n < CP / 8; ++n)
            store_pair(exact, n * 8 + 2 * t, a.channels, (acc[n][2 * r] + fine[n][2 * r]) * inv,
                       (acc[n][2 * r + 1] + fine[n][2 * r + 1]) * inv, false);
        }
        // An empty row keeps +inf: its probabilities come out as 0 in the backward pass.
        if (a.lse != nullptr && t == 0)
          a.lse[int64_t(row) * a.heads + span.h0 + head] = sum[r] == 0.0f ? INFINITY : fmaf(top[r], unit, log2f(sum[r]));
      }
    } else if (a.grad_q != nullptr) {
      const float back = a.scale / lift;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = s_qrows[half * 16 + g + 8 * r];
        if (row < 0) continue;
        T* out = static_cast<T*>(a.grad_q) + (int64_t(row) * a.heads + span.h0 + head) * a.channels;
#pragma unroll
        for (int n = 0; n < CP / 8; ++n)
          store_pair(out, n * 8 + 2 * t, a.channels, acc[n][2 * r] * back, acc[n][2 * r + 1] * back, a.wide_out);
      }
    }
  }
  if constexpr (BACK) {
    if (bias && a.table_part != nullptr) {
      // Each thread summed into a column of its own: lanes, then the head's two warps, in a fixed order.
      __syncthreads();
      for (int b = 0; b < a.buckets; ++b) {
        float x = s_hist[b * blockDim.x + tid];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(kFullMask, x, d);
        if (lane == 0) s_hist[b * blockDim.x + tid] = x;
      }
      __syncthreads();
      for (int i = tid; i < span.heads * a.buckets; i += blockDim.x) {
        const int h = i / a.buckets, b = i % a.buckets;
        const float x = s_hist[b * blockDim.x + h * 64] + s_hist[b * blockDim.x + h * 64 + 32];
        a.table_part[(tile * a.heads + span.h0) * a.buckets + i] = x / lift;
      }
    }
  }
}

template <typename T, int CP, bool BACK, bool EXACT>
cudaError_t run_query_tile(const AttendArgs& a, cudaStream_t stream) {
  const QueryTileSmem s =
      query_tile_smem(sizeof(T), CP, a.kv_cta, a.heads_cta, BACK, a.table != nullptr, a.buckets);
  cudaError_t e = allow_smem(k_query_tile<T, CP, BACK, EXACT>, s.total);
  if (e != cudaSuccess) return e;
  const unsigned groups = a.heads_cta >= a.group
                              ? unsigned((a.kv_heads + a.kv_cta - 1) / a.kv_cta)
                              : unsigned(a.kv_heads) * unsigned((a.group + a.heads_cta - 1) / a.heads_cta);
  const dim3 grid(unsigned(a.map.num_tiles), groups, BACK ? 1 : unsigned(a.splits));
  k_query_tile<T, CP, BACK, EXACT><<<grid, a.heads_cta * 64, s.total, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, bool BACK, bool EXACT>
cudaError_t run_query_tile_by_channels(const AttendArgs& a, cudaStream_t stream) {
  switch (padded_channels(a.channels)) {
    case 32: return run_query_tile<T, 32, BACK, EXACT>(a, stream);
    case 64: return run_query_tile<T, 64, BACK, EXACT>(a, stream);
    case 96: return run_query_tile<T, 96, BACK, EXACT>(a, stream);
    default: return run_query_tile<T, 128, BACK, EXACT>(a, stream);
  }
}

template <bool BACK, bool EXACT>
cudaError_t run_query_tile_by_type(const AttendArgs& a, int dtype, cudaStream_t stream) {
  if (dtype == TBVH_BF16) return run_query_tile_by_channels<__nv_bfloat16, BACK, EXACT>(a, stream);
  if (dtype == TBVH_F16) return run_query_tile_by_channels<__half, BACK, EXACT>(a, stream);
  if constexpr (!EXACT) return run_query_tile_by_channels<float, BACK, false>(a, stream);
  return cudaErrorInvalidValue;
}

}  // namespace tbvh
