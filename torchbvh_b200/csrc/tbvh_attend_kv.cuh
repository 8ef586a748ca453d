// Block attention by key block: the part of the backward pass that sums over
// queries.
//
//   p = 2^(z - m - log2 l), dS = p (V dO^T - <dO, O>)  (rows: keys, columns: queries)
//   dV = sum p dO;  dK = scale sum dS Q
//
// A thread block serves one block of 64 keys and one key/value head; four warps,
// 16 keys each. It walks the block's list of queries, 32 a step: only those that
// selected it, so no score is computed in vain, in ascending order, so the sums
// run in a fixed order without atomics, and over the query heads that share the
// key/value head. Every key row belongs to exactly one block, so every gradient
// row is written once, also for blocks that nobody selected.
//
// Two or four key/value heads a thread block would share a step's buckets, but
// one, and more thread blocks an SM, was faster (16,384 queries, 8 heads of 32,
// bf16, the whole training pass: 1.06 ms for one, 1.10 for two, 1.19 for four; 2
// heads of 64 shared by 8: 0.86, 0.99 and 1.16).
//
// Bound by issue and latency as the query tiles' kernel, and by its longest lists: 0.43
// ms of that training pass, issue slots 52 % busy while an SM has work and 24 % of all
// cycles, matrix pipe 17 %, DRAM 1 %. A list is one thread block's work; of those 256 the
// mean has 512 queries and the longest some 5,000 (a run of leaves that straddles large
// cells of the order has a large box, in which many queries lie). 3 x 1,999 queries, 3
// heads of 20, float32: mean 250, longest 1,200 to 1,600, 0.23 ms, 15 % of all cycles.
#pragma once

#include "tbvh_attend.cuh"

namespace tbvh {

struct KeyBlockSmem {
  uint32_t bias, k, v, q, d, stats, delta, rows, krows, buckets, pts, kpts, table, total;
};

constexpr int kKeyBucketRow = kTileQueries + 8;  // bytes of a key's row of buckets

__host__ __device__ inline KeyBlockSmem key_block_smem(int size, int cp, int group, bool bias) {
  KeyBlockSmem s{};
  const uint32_t row = uint32_t(cp * size + 16);
  uint32_t at = 0;
  auto take = [&](uint32_t bytes) {
    const uint32_t was = at;
    at += (bytes + 15) / 16 * 16;
    return was;
  };
  if (bias) s.bias = take(group * kMaxBuckets * 4);
  s.k = take(kBlockLeaves * row);
  s.v = take(kBlockLeaves * row);
  s.q = take(2 * kTileQueries * row);
  s.d = take(2 * kTileQueries * row);
  s.stats = take(2 * kTileQueries * 8);
  s.delta = take(2 * kTileQueries * 4);
  s.rows = take(2 * kTileQueries * 4);
  s.krows = take(kBlockLeaves * 4);
  if (bias) {
    s.buckets = take(2 * kBlockLeaves * kKeyBucketRow);
    s.pts = take(2 * 3 * kTileQueries * 4);
    s.kpts = take(4 * kBlockLeaves * 4);
    s.table = take(sizeof(BucketTable));
  }
  s.total = at;
  return s;
}

template <typename T, int CP>
__global__ void __launch_bounds__(128, CP <= 32 && sizeof(T) == 2 ? 4 : CP <= 64 ? 3 : 2)
    k_key_block(AttendArgs a) {
  using F = Frag<T>;
  constexpr uint32_t SIZE = sizeof(T);
  constexpr int NT = kTileQueries / 8;
  constexpr bool HELD = sizeof(T) == 2 && CP <= 64;
  constexpr int HOLD = HELD ? CP / F::STEP : 1;
  extern __shared__ __align__(256) char smem[];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Crew crew{tid, int(blockDim.x)};
  const int64_t block = blockIdx.x;
  const int kv = blockIdx.y;
  const BlockCloud c = a.map.of_block(block);
  const bool bias = a.table != nullptr;
  const KeyBlockSmem off = key_block_smem(sizeof(T), CP, a.group, bias);
  const uint32_t base = smem_u32(smem);
  float2* s_stats = reinterpret_cast<float2*>(smem + off.stats);
  float* s_delta = reinterpret_cast<float*>(smem + off.delta);
  int* s_rows = reinterpret_cast<int*>(smem + off.rows);
  int* s_krows = reinterpret_cast<int*>(smem + off.krows);
  float* s_bias = reinterpret_cast<float*>(smem + off.bias);
  uint8_t* s_buckets = reinterpret_cast<uint8_t*>(smem + off.buckets);
  float* s_pts = reinterpret_cast<float*>(smem + off.pts);
  float4* s_kpts = reinterpret_cast<float4*>(smem + off.kpts);  // negated
  BucketTable& s_table = *reinterpret_cast<BucketTable*>(smem + off.table);
  const uint32_t rs = row_bytes<T, CP>(1);
  const uint32_t stage = kTileQueries * rs;

  const int64_t begin = a.plan.query_begin[block];
  const int listed = int(a.plan.query_begin[block + 1] - begin);
  const int chunks = (listed + kTileQueries - 1) / kTileQueries;
  const uint32_t* list = a.plan.list + begin;
  const int64_t leaf0 = (block - c.b0) * kBlockLeaves;
  const int valid = c.n - leaf0 < kBlockLeaves ? int(c.n - leaf0) : kBlockLeaves;
  // Steps: every chunk once for each query head that shares the key/value head.
  const int group = a.group;
  const int64_t steps = int64_t(chunks) * group;
  const Units units(a.scale);

  if (tid < kBlockLeaves) {
    s_krows[tid] = key_row(a, c, leaf0 + tid);
    if (bias) {
      const float* p = a.aabbs + (leaf_row0(c) + leaf0 + tid) * 2 * a.dim;
      s_kpts[tid] = tid < valid ? make_float4(-p[0], -p[1], a.dim == 3 ? -p[2] : 0.0f, 0.0f) : make_float4(0, 0, 0, 0);
    }
  }
  // The warps take turns, a chunk each: a chunk's warp asks for its list elements
  // three chunks ahead, for their rows and points two chunks ahead (one query a
  // lane), and copies the rows one step ahead.
  const bool whole = a.width == 16 && a.channels == CP;
  const int row_words = a.heads * CP * int(SIZE) / 16;
  const int warps = int(blockDim.x) / 32;
  uint32_t next_slot = 0;
  int next_row = 0;
  float next_pt[3] = {0.0f, 0.0f, 0.0f};
  auto ask_list = [&](int e) { next_slot = list[min(e * kTileQueries + lane, listed - 1)]; };
  auto ask_rows = [&]() {
    next_row = a.plan.query_row[next_slot];
    if (bias) {
      const float* p =
          a.plan.query_point + int64_t(next_slot / kTileQueries) * 3 * kTileQueries + next_slot % kTileQueries;
      for (int x = 0; x < 3; ++x) next_pt[x] = p[x * kTileQueries];
    }
  };
  auto put = [&](int e) {
    s_rows[(e & 1) * kTileQueries + lane] = next_row;
    if (bias)
      for (int x = 0; x < 3; ++x) s_pts[((e & 1) * 3 + x) * kTileQueries + lane] = next_pt[x];
  };
  auto copy = [&](int64_t step, int e, int member) {  // step = e * group + member, by one warp (or all)
    const int slot = int(step & 1);
    const int* rows = s_rows + (e & 1) * kTileQueries;
    const int head = kv * group + member;
    const uint32_t to = base + slot * stage;
    if (whole) {
      const int64_t begin = int64_t(head) * CP * SIZE;
      copy_words(to + off.q, to + off.d, static_cast<const char*>(a.q) + begin,
                 static_cast<const char*>(a.grad_out) + begin, uint32_t(rows[lane]) * row_words, CP * int(SIZE) / 16, rs,
                 lane);
    } else {
      auto row_of = [&](int r) { return rows[r]; };
      const Rows<T, CP> q{static_cast<const T*>(a.q), a.heads, a.channels, head, 1, a.width, rs};
      const Rows<T, CP> d{static_cast<const T*>(a.grad_out), a.heads, a.channels, head, 1, a.width, rs};
      q.copy(to + off.q, kTileQueries, row_of, crew);
      d.copy(to + off.d, kTileQueries, row_of, crew);
      if (warp != 0) return;
    }
    const int64_t at = int64_t(rows[lane]) * a.heads + head;
    float2* stats = s_stats + slot * kTileQueries + lane;
    // Past the list's end the sum is infinite: p = 0.
    if (e * kTileQueries + lane < listed) cp_async<8>(smem_u32(stats), a.stats_in + at, true);
    else *stats = make_float2(0.0f, INFINITY);
    cp_async<4>(smem_u32(s_delta + slot * kTileQueries + lane), a.delta + at, true);
  };
  auto sort_pairs = [&](int e) {  // distance buckets of chunk e
    if (bias && e < chunks) {
      const int slot = e & 1;
      uint8_t* to = s_buckets + slot * kBlockLeaves * kKeyBucketRow;
      const float* p = s_pts + slot * 3 * kTileQueries;
      if (s_table.crowded) sort_step<true>(to, kKeyBucketRow, s_table, s_kpts, kBlockLeaves, p, ~0u);
      else sort_step<false>(to, kKeyBucketRow, s_table, s_kpts, kBlockLeaves, p, ~0u);
    }
  };

  clear_padding<T, CP>(smem + off.k, rs, kBlockLeaves, 1, a.channels, crew);
  clear_padding<T, CP>(smem + off.v, rs, kBlockLeaves, 1, a.channels, crew);
  clear_padding<T, CP>(smem + off.q, rs, 2 * kTileQueries, 1, a.channels, crew);
  clear_padding<T, CP>(smem + off.d, rs, 2 * kTileQueries, 1, a.channels, crew);
  if (bias)
    for (int i = tid; i < group * a.buckets; i += blockDim.x)
      s_bias[(i / a.buckets) * kMaxBuckets + i % a.buckets] = units.of_bias(a.table[int64_t(kv) * group * a.buckets + i]);
  if (warp < 2 && warp < chunks) {
    ask_list(warp);
    ask_rows();
    put(warp);
  }
  if (chunks > 2 && warp == 2 % warps) ask_list(2);
  __syncthreads();
  {
    auto row_of = [&](int r) { return s_krows[r]; };
    const Rows<T, CP> keys{static_cast<const T*>(a.k), a.kv_heads, a.channels, kv, 1, a.width, rs};
    const Rows<T, CP> values{static_cast<const T*>(a.v), a.kv_heads, a.channels, kv, 1, a.width, rs};
    keys.copy(base + off.k, kBlockLeaves, row_of, crew);
    values.copy(base + off.v, kBlockLeaves, row_of, crew);
  }
  if (chunks > 0 && (!whole || warp == 0)) copy(0, 0, 0);
  cp_commit();
  if (bias) {
    s_table.make(a.edges, a.buckets - 1);
    __syncthreads();
  }
  sort_pairs(0);
  cp_wait<0>();
  __syncthreads();

  const bool mine = warp * 16 < valid;
  const int g = lane >> 2, t = lane & 3;
  // Byte addresses with the lane's offset; query tiles of stage 0.
  const uint32_t k_at = base + off.k + warp * 16 * rs + F::lane_a(rs, lane), v_at = k_at + (off.v - off.k);
  const uint32_t nk = F::lane_nk(rs, lane), kn = F::lane_kn(rs, lane);
  const uint8_t* near0 = s_buckets + (warp * 16 + g) * kKeyBucketRow + 8 * t;
  const float lift = gradient_lift<T>(a), unit = units.unit;
  typename F::A held_k[HOLD], held_v[HOLD];
  if constexpr (HELD) {
    if (mine) {
      hold<T, CP>(held_k, k_at, rs);
      hold<T, CP>(held_v, v_at, rs);
    }
  }
  float dk[CP / 8][4] = {}, dv[CP / 8][4] = {};

  int e = 0, member = 0;
  for (int64_t step = 0; step < steps; ++step) {
    cp_wait<0>();
    __syncthreads();
    const bool last = member + 1 == group;  // of this entry
    if (step + 1 < steps && (!whole || warp == (last ? (e + 1) % warps : e % warps)))
      copy(step + 1, last ? e + 1 : e, last ? 0 : member + 1);
    cp_commit();
    if (member == 0) sort_pairs(e + 1);
    const bool asked = last && e + 2 < chunks && warp == (e + 2) % warps;
    if (asked) ask_rows();
    if (last && e + 3 < chunks && warp == (e + 3) % warps) ask_list(e + 3);
    if (mine) {
      const int slot = int(step & 1);
      const uint32_t q_at = base + off.q + slot * stage, d_at = base + off.d + slot * stage;
      const float2* stats = s_stats + slot * kTileQueries + 2 * t;
      const float* delta = s_delta + slot * kTileQueries + 2 * t;
      const uint32_t head_bias = base + off.bias + member * kMaxBuckets * 4;
      float s[NT][4], ds[NT][4];
      const uint8_t* near = near0 + (e & 1) * kBlockLeaves * kKeyBucketRow;
      if (bias)
        logits<T, CP, HELD, true, false>(s, held_k, k_at, rs, q_at + nk, rs, head_bias, near, 8 * kKeyBucketRow,
                                         a.scale * kLog2e, units.folded);
      else
        logits<T, CP, HELD, false, false>(s, held_k, k_at, rs, q_at + nk, rs, head_bias, near, 8 * kKeyBucketRow,
                                          a.scale * kLog2e, units.folded);
      multiply_nk<T, CP, NT, HELD, true>(ds, held_v, v_at, rs, d_at + nk, rs);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float4 m = *reinterpret_cast<const float4*>(stats + n * 8);
        const float2 d = *reinterpret_cast<const float2*>(delta + n * 8);
        const Pair minus_top = pair(-m.x, -m.z), minus_logsum = pair(-m.y, -m.w), minus_d = pair(-d.x, -d.y);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const Pair z = add2(pair(s[n][2 * r], s[n][2 * r + 1]), minus_top);
          const float2 x = unpair(fma2(z, both(unit), minus_logsum));
          s[n][2 * r] = exp2_fast(x.x);
          s[n][2 * r + 1] = exp2_fast(x.y);
          Pair y = add2(pair(ds[n][2 * r], ds[n][2 * r + 1]), minus_d);
          if constexpr (SIZE == 2) y = mul2(y, both(lift));
          Pair p = pair(s[n][2 * r], s[n][2 * r + 1]);
          y = mul2(p, y);
          ds[n][2 * r] = unpair(y).x;
          ds[n][2 * r + 1] = unpair(y).y;
          if constexpr (F::PEAK != 1.0f) p = mul2(p, both(F::PEAK));
          s[n][2 * r] = unpair(p).x;
          s[n][2 * r + 1] = unpair(p).y;
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
            F::pair_kn(b, d_at + kn + st * F::STEP * rs + j * 16 * SIZE, rs);
            F::mma(dv[2 * j], p, b[0], b[1]);
            F::mma(dv[2 * j + 1], p, b[2], b[3]);
            F::pair_kn(b, q_at + kn + st * F::STEP * rs + j * 16 * SIZE, rs);
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
            F::pair_kn(b, d_at + kn + st * F::STEP * rs + j * 16 * SIZE, rs);
            F::mma(part_v[0], p, b[0], b[1]);
            F::mma(part_v[1], p, b[2], b[3]);
            F::pair_kn(b, q_at + kn + st * F::STEP * rs + j * 16 * SIZE, rs);
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
    if (asked) put(e + 2);  // its slot held chunk e's rows, which nothing copies any more
    if (last) {
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
      const int row = s_krows[warp * 16 + g + 8 * r];
      if (row < 0) continue;
      const int64_t at = (int64_t(row) * a.kv_heads + kv) * a.channels;
      T* out_k = static_cast<T*>(a.grad_k) + at;
      T* out_v = static_cast<T*>(a.grad_v) + at;
#pragma unroll
      for (int n = 0; n < CP / 8; ++n) {
        store_pair(out_k, n * 8 + 2 * t, a.channels, dk[n][2 * r] * back, dk[n][2 * r + 1] * back, a.wide_out);
        store_pair(out_v, n * 8 + 2 * t, a.channels, dv[n][2 * r] / F::PEAK, dv[n][2 * r + 1] / F::PEAK, a.wide_out);
      }
    }
  }
}

template <typename T, int CP>
cudaError_t run_key_block(const AttendArgs& a, cudaStream_t stream) {
  const KeyBlockSmem s = key_block_smem(sizeof(T), CP, a.group, a.table != nullptr);
  const cudaError_t e = allow_smem(k_key_block<T, CP>, s.total);
  if (e != cudaSuccess) return e;
  const dim3 grid(unsigned(a.map.num_blocks), unsigned(a.kv_heads));
  k_key_block<T, CP><<<grid, 128, s.total, stream>>>(a);
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
