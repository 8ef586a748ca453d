// Block attention by key block: the part of the backward pass that sums over
// queries.
//
//   p = 2^(z - lse), dS = p (V dO^T - <dO, O>)  (rows: keys, columns: queries)
//   dV = sum p dO;  dK = scale sum dS Q
//
// A thread block serves one block of 64 keys and up to two key/value heads;
// four warps a head, 16 keys each. It walks the block's list of queries, 32 a
// step: only those that selected it, so no score is computed in vain, in
// ascending order, so the sums run in a fixed order without atomics, and over
// the query heads that share a key/value head. Every key row belongs to exactly
// one block, so every gradient row is written once, also for blocks that nobody
// selected.
#pragma once

#include "tbvh_attend.cuh"

namespace tbvh {

constexpr int kKvHeads = 2;  // key/value heads of one thread block, at most

struct KeyBlockSmem {
  uint32_t k, v, q, d, lse, delta, rows, krows, bias, buckets, pts, kpts, table, total;
};

__host__ __device__ inline KeyBlockSmem key_block_smem(int size, int cp, int kvs, int group, bool bias) {
  KeyBlockSmem s{};
  const uint32_t ld = uint32_t(cp + 16 / size);
  uint32_t at = 0;
  auto take = [&](uint32_t bytes) {
    const uint32_t was = at;
    at += (bytes + 15) / 16 * 16;
    return was;
  };
  s.k = take(kvs * kBlockLeaves * ld * size);
  s.v = take(kvs * kBlockLeaves * ld * size);
  s.q = take(2 * kvs * kTileQueries * ld * size);
  s.d = take(2 * kvs * kTileQueries * ld * size);
  s.lse = take(2 * kvs * kTileQueries * 4);
  s.delta = take(2 * kvs * kTileQueries * 4);
  s.rows = take(2 * kTileQueries * 4);
  s.krows = take(kBlockLeaves * 4);
  if (bias) {
    s.bias = take(kvs * group * kMaxBuckets * 4);
    s.buckets = take(2 * kBlockLeaves * (kTileQueries + 4));
    s.pts = take(2 * 3 * kTileQueries * 4);
    s.kpts = take(3 * kBlockLeaves * 4);
    s.table = take(sizeof(BucketTable));
  }
  s.total = at;
  return s;
}

template <typename T, int CP>
__global__ void __launch_bounds__(256) k_key_block(AttendArgs a) {
  using F = Frag<T>;
  constexpr int LD = Tile<T, CP>::LD;
  constexpr int NT = kTileQueries / 8;
  constexpr bool HELD = sizeof(T) == 2 && CP <= 64;
  constexpr int HOLD = HELD ? CP / F::STEP : 1;
  constexpr int BROW = kTileQueries + 4;
  extern __shared__ __align__(16) char smem[];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t block = blockIdx.x;
  const int kv0 = blockIdx.y * a.kv_cta;
  const int kvs = min(a.kv_cta, a.kv_heads - kv0);
  const BlockCloud c = a.map.of_block(block);
  const bool bias = a.table != nullptr;
  const KeyBlockSmem off = key_block_smem(sizeof(T), CP, a.kv_cta, a.group, bias);
  T* s_k = reinterpret_cast<T*>(smem + off.k);
  T* s_v = reinterpret_cast<T*>(smem + off.v);
  T* s_q = reinterpret_cast<T*>(smem + off.q);
  T* s_d = reinterpret_cast<T*>(smem + off.d);
  float* s_lse = reinterpret_cast<float*>(smem + off.lse);
  float* s_delta = reinterpret_cast<float*>(smem + off.delta);
  int* s_rows = reinterpret_cast<int*>(smem + off.rows);
  int* s_krows = reinterpret_cast<int*>(smem + off.krows);
  float* s_bias = reinterpret_cast<float*>(smem + off.bias);
  uint8_t* s_buckets = reinterpret_cast<uint8_t*>(smem + off.buckets);
  float* s_pts = reinterpret_cast<float*>(smem + off.pts);
  float* s_kpts = reinterpret_cast<float*>(smem + off.kpts);
  BucketTable& s_table = *reinterpret_cast<BucketTable*>(smem + off.table);
  const int k_tile = kBlockLeaves * LD, q_tile = kTileQueries * LD;
  const int stage = a.kv_cta * q_tile;

  const int64_t begin = a.plan.query_begin[block];
  const int listed = int(a.plan.query_begin[block + 1] - begin);
  const int chunks = (listed + kTileQueries - 1) / kTileQueries;
  const uint32_t* list = a.plan.list + begin;
  const int64_t leaf0 = (block - c.b0) * kBlockLeaves;
  const int valid = c.n - leaf0 < kBlockLeaves ? int(c.n - leaf0) : kBlockLeaves;
  // Steps: every chunk once for each query head that shares a key/value head.
  const int group = a.group;
  const int64_t steps = int64_t(chunks) * group;
  // As in the query-tile kernel.
  const bool folded = a.scale >= 0x1p-30f && a.scale <= 0x1p30f;
  const float unit = folded ? a.scale * kLog2e : 1.0f;
  const float bias_unit = folded ? 1.0f / a.scale : kLog2e;

  if (tid < kBlockLeaves) {
    s_krows[tid] = key_row(a, c, leaf0 + tid);
    if (bias) {
      const float* p = a.aabbs + (leaf_row0(c) + leaf0 + tid) * 2 * a.dim;
      for (int x = 0; x < 3; ++x) s_kpts[x * kBlockLeaves + tid] = tid < valid && x < a.dim ? p[x] : 0.0f;
    }
  }
  int next_row = -1;
  float next_pt[3] = {0.0f, 0.0f, 0.0f};
  auto fetch = [&](int e) {
    if (tid < kTileQueries && e < chunks) {
      const int at = e * kTileQueries + tid;
      next_row = -1;
      if (at < listed) {
        const uint32_t slot = list[at];
        next_row = a.plan.query_row[slot];
        if (bias)
          for (int x = 0; x < 3; ++x)
            next_pt[x] = a.plan.query_point[(int64_t(slot / kTileQueries) * 3 + x) * kTileQueries + slot % kTileQueries];
      }
    }
  };
  auto put = [&](int e) {
    if (tid < kTileQueries && e < chunks) {
      const int slot = e & 1;
      s_rows[slot * kTileQueries + tid] = next_row;
      if (bias)
        for (int x = 0; x < 3; ++x) s_pts[(slot * 3 + x) * kTileQueries + tid] = next_pt[x];
    }
  };
  auto copy = [&](int64_t step, int e, int member) {  // step = e * group + member
    if (step < steps) {
      const int slot = int(step & 1);
      const int* rows = s_rows + (e & 1) * kTileQueries;
      // Query heads kv * group + member, one a key/value head.
      copy_rows<T, CP>(s_q + slot * stage, q_tile, static_cast<const T*>(a.q), rows, kTileQueries, a.heads, a.channels,
                       kv0 * group + member, kvs, a.width, group);
      copy_rows<T, CP>(s_d + slot * stage, q_tile, static_cast<const T*>(a.grad_out), rows, kTileQueries, a.heads,
                       a.channels, kv0 * group + member, kvs, a.width, group);
      for (int i = tid; i < kvs * kTileQueries; i += blockDim.x) {
        const int h = i / kTileQueries, q = i % kTileQueries, row = rows[q];
        const int64_t at = int64_t(row < 0 ? 0 : row) * a.heads + (kv0 + h) * group + member;
        float* lse = s_lse + (slot * a.kv_cta + h) * kTileQueries + q;
        // Past the list's end the rows are zeros and the sum is infinite: p = 0.
        if (row >= 0) cp_async<4>(smem_u32(lse), a.lse_in + at, true);
        else *lse = INFINITY;
        cp_async<4>(smem_u32(s_delta + (slot * a.kv_cta + h) * kTileQueries + q), a.delta + at, row >= 0);
      }
    }
    cp_commit();
  };
  // Distance buckets of chunk e, times four: a thread has a key and four neighbouring queries.
  auto sort_pairs = [&](int e) {
    if (bias && e < chunks) {
      const int slot = e & 1;
      for (int u = tid; u < kTileQueries * kBlockLeaves / 4; u += blockDim.x) {
        const int key = u / (kTileQueries / 4), q4 = u % (kTileQueries / 4) * 4;
        const float kx = s_kpts[key], ky = s_kpts[kBlockLeaves + key], kz = s_kpts[2 * kBlockLeaves + key];
        const float* p = s_pts + slot * 3 * kTileQueries + q4;
        const float4 px = *reinterpret_cast<const float4*>(p);
        const float4 py = *reinterpret_cast<const float4*>(p + kTileQueries);
        const float4 pz = *reinterpret_cast<const float4*>(p + 2 * kTileQueries);
        const bool three = a.dim == 3;
        const uint32_t b0 = s_table.find(pair_distance(px.x, py.x, pz.x, kx, ky, kz, three));
        const uint32_t b1 = s_table.find(pair_distance(px.y, py.y, pz.y, kx, ky, kz, three));
        const uint32_t b2 = s_table.find(pair_distance(px.z, py.z, pz.z, kx, ky, kz, three));
        const uint32_t b3 = s_table.find(pair_distance(px.w, py.w, pz.w, kx, ky, kz, three));
        *reinterpret_cast<uint32_t*>(s_buckets + (slot * kBlockLeaves + key) * BROW + q4) =
            (b0 | b1 << 8 | b2 << 16 | b3 << 24) << 2;
      }
    }
  };

  clear_padding<T, CP>(s_k, a.kv_cta * kBlockLeaves, a.channels);
  clear_padding<T, CP>(s_v, a.kv_cta * kBlockLeaves, a.channels);
  clear_padding<T, CP>(s_q, 2 * a.kv_cta * kTileQueries, a.channels);
  clear_padding<T, CP>(s_d, 2 * a.kv_cta * kTileQueries, a.channels);
  fetch(0);
  put(0);
  if (bias) {
    for (int i = tid; i < kvs * group * a.buckets; i += blockDim.x)
      s_bias[(i / a.buckets) * kMaxBuckets + i % a.buckets] = a.table[int64_t(kv0) * group * a.buckets + i] * bias_unit;
  }
  __syncthreads();
  copy_rows<T, CP>(s_k, k_tile, static_cast<const T*>(a.k), s_krows, kBlockLeaves, a.kv_heads, a.channels, kv0, kvs,
                   a.width);
  copy_rows<T, CP>(s_v, k_tile, static_cast<const T*>(a.v), s_krows, kBlockLeaves, a.kv_heads, a.channels, kv0, kvs,
                   a.width);
  copy(0, 0, 0);
  fetch(1);
  put(1);
  if (bias) {
    s_table.make(a.edges, a.buckets - 1);
    __syncthreads();
  }
  sort_pairs(0);
  cp_wait<0>();
  __syncthreads();

  const int kv = warp >> 2, quarter = warp & 3;
  const bool mine = kv < kvs && quarter * 16 < valid;
  const int g = lane >> 2, t = lane & 3;
  const T* k_rows = s_k + kv * k_tile;
  const T* v_rows = s_v + kv * k_tile;
  const float lift = gradient_lift<T>(a);
  typename F::A held_k[HOLD], held_v[HOLD];
  if constexpr (HELD) {
    if (mine) {
      hold<T, CP>(held_k, k_rows, quarter * 16, lane);
      hold<T, CP>(held_v, v_rows, quarter * 16, lane);
    }
  }
  float dk[CP / 8][4] = {}, dv[CP / 8][4] = {};

  int e = 0, member = 0;
  for (int64_t step = 0; step < steps; ++step) {
    cp_wait<0>();
    __syncthreads();
    const bool last = member + 1 == group;  // of this entry
    copy(step + 1, last ? e + 1 : e, last ? 0 : member + 1);
    if (member == 0) {
      sort_pairs(e + 1);
      fetch(e + 2);
    }
    if (mine) {
      const int slot = int(step & 1);
      const T* q_rows = s_q + slot * stage + kv * q_tile;
      const T* d_rows = s_d + slot * stage + kv * q_tile;
      const float* lse = s_lse + (slot * a.kv_cta + kv) * kTileQueries + 2 * t;
      const float* delta = s_delta + (slot * a.kv_cta + kv) * kTileQueries + 2 * t;
      const char* head_bias = reinterpret_cast<const char*>(s_bias + (kv * group + member) * kMaxBuckets);
      const uint8_t* near = s_buckets + ((e & 1) * kBlockLeaves + quarter * 16 + g) * BROW + 2 * t;
      float s[NT][4], ds[NT][4] = {};
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
        multiply_nk<T, CP, NT, HELD>(s, held_k, k_rows, quarter * 16, q_rows, 0, lane);
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
        multiply_nk<T, CP, NT, HELD>(s, held_k, k_rows, quarter * 16, q_rows, 0, lane);
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
      multiply_nk<T, CP, NT, HELD>(ds, held_v, v_rows, quarter * 16, d_rows, 0, lane);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 l = *reinterpret_cast<const float2*>(lse + n * 8);
        const float2 d = *reinterpret_cast<const float2*>(delta + n * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[n][j] = exp2_fast(fmaf(s[n][j], unit, -((j & 1) ? l.y : l.x)));
          ds[n][j] = s[n][j] * (lift * (ds[n][j] - ((j & 1) ? d.y : d.x)));
        }
      }
      constexpr int STEPS = kTileQueries / F::STEP;
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          typename F::A p, x;
          from_acc<T>(p, s, st);
          from_acc<T>(x, ds, st);
#pragma unroll
          for (int j = 0; j < CP / 16; ++j) {
            typename F::B b;
            F::pair_kn(b, d_rows, LD, st * F::STEP, j * 16, lane);
            F::mma(dv[2 * j], p, b[0], b[1]);
            F::mma(dv[2 * j + 1], p, b[2], b[3]);
            F::pair_kn(b, q_rows, LD, st * F::STEP, j * 16, lane);
            F::mma(dk[2 * j], x, b[0], b[1]);
            F::mma(dk[2 * j + 1], x, b[2], b[3]);
          }
        }
      } else {
        // The matrix pipe truncates as it adds: over a long list that would cost
        // float32 its last bits, so each entry's products are summed by
        // themselves and added with rounding.
#pragma unroll
        for (int j = 0; j < CP / 16; ++j) {
          float part_v[2][4] = {}, part_k[2][4] = {};
#pragma unroll
          for (int st = 0; st < STEPS; ++st) {
            typename F::A p, x;
            from_acc<T>(p, s, st);
            from_acc<T>(x, ds, st);
            typename F::B b;
            F::pair_kn(b, d_rows, LD, st * F::STEP, j * 16, lane);
            F::mma(part_v[0], p, b[0], b[1]);
            F::mma(part_v[1], p, b[2], b[3]);
            F::pair_kn(b, q_rows, LD, st * F::STEP, j * 16, lane);
            F::mma(part_k[0], x, b[0], b[1]);
            F::mma(part_k[1], x, b[2], b[3]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dv[2 * j][i] += part_v[0][i];
            dv[2 * j + 1][i] += part_v[1][i];
            dk[2 * j][i] += part_k[0][i];
            dk[2 * j + 1][i] += part_k[1][i];
          }
        }
      }
    }
    if (last) {
      put(e + 2);  // its slot holds this entry's rows, which the next step's copies were the last to read
      ++e;
      member = 0;
    } else {
      ++member;
    }
  }

  if (mine) {
    const float back = a.scale / lift;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = s_krows[quarter * 16 + g + 8 * r];
      if (row < 0) continue;
      const int64_t at = (int64_t(row) * a.kv_heads + kv0 + kv) * a.channels;
      T* out_k = static_cast<T*>(a.grad_k) + at;
      T* out_v = static_cast<T*>(a.grad_v) + at;
#pragma unroll
      for (int n = 0; n < CP / 8; ++n) {
        store_pair(out_k, n * 8 + 2 * t, a.channels, dk[n][2 * r] * back, dk[n][2 * r + 1] * back, a.wide_out);
        store_pair(out_v, n * 8 + 2 * t, a.channels, dv[n][2 * r], dv[n][2 * r + 1], a.wide_out);
      }
    }
  }
}

template <typename T, int CP>
cudaError_t run_key_block(AttendArgs a, cudaStream_t stream) {
  a.kv_cta = a.kv_heads < kKvHeads ? a.kv_heads : kKvHeads;
  KeyBlockSmem s = key_block_smem(sizeof(T), CP, a.kv_cta, a.group, a.table != nullptr);
  if (s.total > 200 * 1024 && a.kv_cta > 1) {
    a.kv_cta = 1;
    s = key_block_smem(sizeof(T), CP, a.kv_cta, a.group, a.table != nullptr);
  }
  const cudaError_t e = allow_smem(k_key_block<T, CP>, s.total);
  if (e != cudaSuccess) return e;
  const dim3 grid(unsigned(a.map.num_blocks), unsigned((a.kv_heads + a.kv_cta - 1) / a.kv_cta));
  k_key_block<T, CP><<<grid, a.kv_cta * 128, s.total, stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_key_block_by_channels(const AttendArgs& a, cudaStream_t stream) {
  switch (padded_channels(a.channels)) {
    case 32: return run_key_block<T, 32>(a, stream);
    case 64: return run_key_block<T, 64>(a, stream);
    case 96: return run_key_block<T, 96>(a, stream);
    default: return run_key_block<T, 128>(a, stream);
  }
}

}  // namespace tbvh
