// Block attention by query tile: the forward pass, and the part of the backward
// pass that sums over keys (gradients of the queries and of the bias table).
//
// A thread block serves one tile (32 queries, neighbours in space) and up to
// four query heads; a warp has one head and 16 of the queries. The block walks
// the tile's entries (64 leaves each, union of what its queries selected): key
// and value rows come by asynchronous copies straight from the caller's order
// (sorted_indices), two stages deep, while the previous entry is computed. A
// query's bit in the entry's mask says whether it takes part; a warp none of
// whose queries does skips the entry. Distance buckets are the same for every
// head: the block computes them once an entry, one byte a pair, and each score
// reads a byte and the head's bias from shared memory.
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
// adding zero products: non-finite keys and values reach only the rows that
// attend to them.
#pragma once

#include "tbvh_attend.cuh"

namespace tbvh {

struct QueryTileSmem {
  uint32_t k, v, q, d, bias, buckets, pts, rows, qpts, qrows, table, hist, total;
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
  s.k = take(2 * kvs * kBlockLeaves * ld * size);
  s.v = take(2 * kvs * kBlockLeaves * ld * size);
  s.q = take(heads * kTileQueries * ld * size);
  s.d = back ? take(heads * kTileQueries * ld * size) : 0;
  s.rows = take(2 * kBlockLeaves * 4);
  s.qrows = take(kTileQueries * 4);
  if (bias) {
    s.bias = take(heads * kMaxBuckets * 4);
    s.buckets = take(2 * kTileQueries * (kBlockLeaves + 4));
    s.pts = take(2 * 3 * kBlockLeaves * 4);
    s.qpts = take(3 * kTileQueries * 4);
    s.table = take(sizeof(BucketTable));
    if (back) s.hist = take(uint32_t(buckets) * heads * 64 * 4);
  }
  s.total = at;
  return s;
}

template <typename T, int CP, bool BACK, bool EXACT>
__global__ void __launch_bounds__(256) k_query_tile(AttendArgs a) {
  using F = Frag<T>;
  constexpr int LD = Tile<T, CP>::LD;
  constexpr int KEYS = BACK ? 32 : 64;  // keys a pass over the registers
  constexpr int NT = KEYS / 8;
  constexpr bool HELD = sizeof(T) == 2 ? (BACK ? CP <= 64 : true) : CP <= 32 && !BACK;
  constexpr int HOLD = HELD ? CP / F::STEP : 1;
  constexpr int BROW = kBlockLeaves + 4;  // bytes of one query's bucket row
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
  float* s_qpts = reinterpret_cast<float*>(smem + off.qpts);
  BucketTable& s_table = *reinterpret_cast<BucketTable*>(smem + off.table);
  float* s_hist = reinterpret_cast<float*>(smem + off.hist);
  const int kv_tile = kBlockLeaves * LD, q_tile = kTileQueries * LD;
  const int stage = a.kv_cta * kv_tile;

  const int all = a.plan.tile_count[tile];
  const int splits = BACK ? 1 : a.splits;
  const int from = int(int64_t(all) * blockIdx.z / splits), count = int(int64_t(all) * (blockIdx.z + 1) / splits) - from;
  const uint2* entries = a.plan.entries + tile * a.plan.capacity + from;
  const int64_t leaves = bias ? leaf_row0(c) : 0;

  if (tid < kTileQueries) {
    s_qrows[tid] = a.plan.query_row[tile * kTileQueries + tid];
    if (bias)
      for (int x = 0; x < 3; ++x)
        s_qpts[x * kTileQueries + tid] = a.plan.query_point[(tile * 3 + x) * kTileQueries + tid];
  }
  // Rows (and points) of entry `e`, one leaf a thread.
  int next_row = -1;
  float next_pt[3] = {0.0f, 0.0f, 0.0f};
  auto fetch = [&](int e) {
    if (tid < kBlockLeaves && e < count) {
      const int64_t leaf = int64_t(entries[e].x) * kBlockLeaves + tid;
      next_row = key_row(a, c, leaf);
      if (bias) {
        const float* p = a.aabbs + (leaves + leaf) * 2 * a.dim;
        for (int x = 0; x < 3; ++x) next_pt[x] = leaf < c.n && x < a.dim ? p[x] : 0.0f;
      }
    }
  };
  auto put = [&](int e) {
    if (tid < kBlockLeaves && e < count) {
      const int slot = e & 1;
      s_rows[slot * kBlockLeaves + tid] = next_row;
      if (bias)
        for (int x = 0; x < 3; ++x) s_pts[(slot * 3 + x) * kBlockLeaves + tid] = next_pt[x];
    }
  };
  auto copy = [&](int e) {
    if (e < count) {
      const int slot = e & 1;
      const int* rows = s_rows + slot * kBlockLeaves;
      copy_rows<T, CP>(s_k + slot * stage, kv_tile, static_cast<const T*>(a.k), rows, kBlockLeaves, a.kv_heads,
                       a.channels, span.kv0, span.kvs, a.width);
      copy_rows<T, CP>(s_v + slot * stage, kv_tile, static_cast<const T*>(a.v), rows, kBlockLeaves, a.kv_heads,
                       a.channels, span.kv0, span.kvs, a.width);
    }
    cp_commit();
  };
  auto sort_pairs = [&](int e) {  // distance buckets of entry e
    if (bias && e < count) {
      const int slot = e & 1;
      const float* p = s_pts + slot * 3 * kBlockLeaves;
      for (int i = tid; i < kTileQueries * kBlockLeaves; i += blockDim.x) {
        const int key = i % kBlockLeaves, q = i / kBlockLeaves;
        const float d = pair_distance(s_qpts[q], s_qpts[kTileQueries + q], s_qpts[2 * kTileQueries + q], p[key],
                                      p[kBlockLeaves + key], p[2 * kBlockLeaves + key], a.dim == 3);
        s_buckets[(slot * kTileQueries + q) * BROW + key] = uint8_t(min(s_table.find(d), a.buckets - 1));
      }
    }
  };

  clear_padding<T, CP>(s_k, 2 * a.kv_cta * kBlockLeaves, a.channels);
  clear_padding<T, CP>(s_v, 2 * a.kv_cta * kBlockLeaves, a.channels);
  clear_padding<T, CP>(s_q, a.heads_cta * kTileQueries, a.channels);
  if constexpr (BACK) clear_padding<T, CP>(s_d, a.heads_cta * kTileQueries, a.channels);
  fetch(0);
  put(0);
  if (bias) {
    for (int i = tid; i < span.heads * a.buckets; i += blockDim.x)
      s_bias[(i / a.buckets) * kMaxBuckets + i % a.buckets] = a.table[int64_t(span.h0) * a.buckets + i] * kLog2e;
    if constexpr (BACK)
      for (int i = tid; i < a.buckets * int(blockDim.x); i += blockDim.x) s_hist[i] = 0.0f;
    s_table.make(a.edges, a.buckets - 1);
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
  sort_pairs(0);
  cp_wait<0>();
  __syncthreads();

  const int head = warp >> 1, half = warp & 1;
  const bool mine = head < span.heads;
  const int kv = mine ? (span.h0 + head) / a.group - span.kv0 : 0;
  const int g = lane >> 2, t = lane & 3;
  const T* q_rows = s_q + head * q_tile;
  const T* d_rows = s_d + head * q_tile;
  const float* head_bias = s_bias + head * kMaxBuckets;
  const float scale = a.scale * kLog2e;

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
    if constexpr (sizeof(T) == 2) {
      if (a.grad_max != nullptr) {
        const float most = __uint_as_float(*a.grad_max);
        if (most > 0.0f && most <= FLT_MAX) lift = exp2f(-floorf(log2f(most)));
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = s_qrows[half * 16 + g + 8 * r];
      if (mine && row >= 0) {
        lse[r] = a.lse_in[int64_t(row) * a.heads + span.h0 + head];
        delta[r] = a.delta[int64_t(row) * a.heads + span.h0 + head] * lift;
      }
    }
  }

  for (int e = 0; e < count; ++e) {
    cp_wait<0>();
    __syncthreads();
    copy(e + 1);
    fetch(e + 2);
    sort_pairs(e + 1);
    const uint2 entry = entries[e];
    const unsigned mask = entry.y >> (half * 16);
    if (mine && (mask & 0xffffu)) {
      const int slot = e & 1;
      const T* k_tile = s_k + slot * stage + kv * kv_tile;
      const T* v_tile = s_v + slot * stage + kv * kv_tile;
      const int64_t left = c.n - int64_t(entry.x) * kBlockLeaves;
      const int valid = left < kBlockLeaves ? int(left) : kBlockLeaves;
      const bool on[2] = {(mask >> g & 1u) != 0, (mask >> (g + 8) & 1u) != 0};
      const uint8_t* near = s_buckets + (slot * kTileQueries + half * 16 + g) * BROW + 2 * t;
#pragma unroll
      for (int k0 = 0; k0 < kBlockLeaves; k0 += KEYS) {
        if (k0 >= valid) break;
        float s[NT][4] = {};
        multiply_nk<T, CP, NT, HELD>(s, held_q, q_rows, half * 16, k_tile, k0, lane);
        // Logits in base 2; -inf where masked.
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int key = k0 + n * 8 + 2 * t;
          float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          if (bias) {
            const uint16_t lo = *reinterpret_cast<const uint16_t*>(near + k0 + n * 8);
            const uint16_t hi = *reinterpret_cast<const uint16_t*>(near + 8 * BROW + k0 + n * 8);
            b[0] = head_bias[lo & 255];
            b[1] = head_bias[lo >> 8];
            b[2] = head_bias[hi & 255];
            b[3] = head_bias[hi >> 8];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[n][i] = on[i >> 1] && key + (i & 1) < valid ? fmaf(s[n][i], scale, b[i]) : -INFINITY;
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
            const float base = most == -INFINITY ? 0.0f : most;  // nothing yet: all p are 0
            shrink[r] = exp2_fast(top[r] - base);
            top[r] = most;
            float add = 0.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                s[n][2 * r + i] = exp2_fast(s[n][2 * r + i] - base);
                add += s[n][2 * r + i];
              }
            }
            sum[r] = sum[r] * shrink[r] + add;
          }
          constexpr int STEPS = KEYS / F::STEP;
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
                F::pair_kn(b, v_tile, LD, k0 + st * F::STEP, (n0 + 2 * j) * 8, lane);
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
              for (int i = 0; i < 4; ++i)
                if (on[i >> 1]) {
                  acc[n0 + j][i] = fmaf(acc[n0 + j][i], shrink[i >> 1], part[j][i]);
                  if constexpr (EXACT) fine[n0 + j][i] = fmaf(fine[n0 + j][i], shrink[i >> 1], low[j][i]);
                }
          }
        } else {
          float ds[NT][4] = {};
          multiply_nk<T, CP, NT, HELD>(ds, held_d, d_rows, half * 16, v_tile, k0, lane);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int key = k0 + n * 8 + 2 * t;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = exp2_fast(s[n][i] - lse[i >> 1]);
              const float grad = p * fmaf(ds[n][i], lift, -delta[i >> 1]);
              ds[n][i] = on[i >> 1] && key + (i & 1) < valid ? grad : 0.0f;
            }
            if (bias) {
              const uint16_t lo = *reinterpret_cast<const uint16_t*>(near + k0 + n * 8);
              const uint16_t hi = *reinterpret_cast<const uint16_t*>(near + 8 * BROW + k0 + n * 8);
              s_hist[(lo & 255) * blockDim.x + tid] += ds[n][0];
              s_hist[(lo >> 8) * blockDim.x + tid] += ds[n][1];
              s_hist[(hi & 255) * blockDim.x + tid] += ds[n][2];
              s_hist[(hi >> 8) * blockDim.x + tid] += ds[n][3];
            }
          }
          constexpr int STEPS = KEYS / F::STEP;
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
                F::pair_kn(b, k_tile, LD, k0 + st * F::STEP, (n0 + 2 * j) * 8, lane);
                F::mma(part[2 * j], p, b[0], b[1]);
                F::mma(part[2 * j + 1], p, b[2], b[3]);
              }
            }
#pragma unroll
            for (int j = 0; j < kChannelGroup; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (on[i >> 1]) acc[n0 + j][i] += part[j][i];
          }
        }
        // (forward) a second pass over the registers starts from the new maximum
      }
    }
    put(e + 2);
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
            part[0] = top[r];
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
          a.lse[int64_t(row) * a.heads + span.h0 + head] = sum[r] == 0.0f ? INFINITY : top[r] + log2f(sum[r]);
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
