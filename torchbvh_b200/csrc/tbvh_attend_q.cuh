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
//   backward   p = 2^(z - m - log2 l), dS = p (dO V^T - <dO, O>)
//              dQ = scale sum dS K;  dT[h][bucket] += dS
//
// EXACT (forward, 16-bit features whose bias table trains): the parts of the
// probabilities that 16 bits do not hold go through products of their own, kept
// apart, so that the output's bits do not depend on them; both sums together are
// the float32 output that <dO, O> is taken from.
//
// A row that did not select the entry keeps its sums by selection, not by
// masking its scores: what it computes there is dropped, so non-finite keys and
// values reach only the rows that attend to them.
//
// Bound by issue and by the latencies between a step's barriers, not by bytes or
// products. 4 x 16,384 queries over 8 blocks, 4 heads of 32, bf16, 32 buckets: 0.34
// ms, 4e11 scores a second (51 TFLOP/s of products), issue slots 58 % busy, matrix
// pipe 14 %, exponentials 17 %, DRAM 2 %; without a bias 0.24 ms. In a training pass
// of 16,384 queries with 8 heads: forward (EXACT) 0.36 ms, backward 0.35 ms.
// Measured and left: rows by bulk copies of one thread (a step 1.7 times as long);
// two warps that share four heads' scores of 16 rows (1.25 to 1.5 times); 32 rows a
// warp (0.35 ms with, 0.24 without a bias).
#pragma once

#include <type_traits>

#include "tbvh_attend.cuh"

namespace tbvh {

constexpr int kStepLeaves = 32;
// Steps whose rows are in shared memory or on their way. Three take the memory of
// a third thread block an SM: 16,384 queries, 8 heads of 32, bf16, with bias, the
// whole training pass 1.23 ms for three and 1.09 for two.
constexpr int kStages = 2;
constexpr int kBucketRow = kStepLeaves + 8;  // bytes of a query's row of buckets

struct QueryTileSmem {
  uint32_t bias, k, v, q, d, places, rows, buckets, pts, qpts, table, hist, total;
};

// Offsets of a thread block's arrays (bias first: its rows lie on 256 bytes).
__host__ __device__ inline QueryTileSmem query_tile_smem(int size, int cp, int kvs, int heads, bool back, bool bias,
                                                         int buckets) {
  QueryTileSmem s{};
  const uint32_t kv_row = uint32_t(kvs * cp * size + 16), q_row = uint32_t(heads * cp * size + 16);
  uint32_t at = 0;
  auto take = [&](uint32_t bytes) {
    const uint32_t was = at;
    at += (bytes + 15) / 16 * 16;
    return was;
  };
  if (bias) s.bias = take(heads * kMaxBuckets * 4);
  s.k = take(kStages * kStepLeaves * kv_row);
  s.v = take(kStages * kStepLeaves * kv_row);
  s.q = take(kTileQueries * q_row);
  s.d = back ? take(kTileQueries * q_row) : 0;
  s.places = take(kStages * kStepLeaves * 4);
  s.rows = take(kTileQueries * 4);
  if (bias) {
    s.buckets = take(2 * kTileQueries * kBucketRow);
    s.pts = take(kStages * 3 * kStepLeaves * 4);
    s.qpts = take(kTileQueries * 16);
    s.table = take(sizeof(BucketTable));
    if (back) s.hist = take(uint32_t(buckets) * heads * 64 * 4);
  }
  s.total = at;
  return s;
}

// Row r of a group of accumulator tiles from n0: old * factor + part where `on`.
template <int N>
__device__ __forceinline__ void keep_group(Pair (&acc)[N][2], int n0, int r, Pair factor,
                                           const float (&part)[kChannelGroup][4], uint32_t on) {
  static_assert(kChannelGroup == 4, "one group is four tiles");
  keep_where(acc[n0][r], acc[n0 + 1][r], acc[n0 + 2][r], acc[n0 + 3][r], factor, pair(part[0][2 * r], part[0][2 * r + 1]),
             pair(part[1][2 * r], part[1][2 * r + 1]), pair(part[2][2 * r], part[2][2 * r + 1]),
             pair(part[3][2 * r], part[3][2 * r + 1]), on);
}

// Registers: with 32 padded channels three blocks of eight warps share an SM.
template <typename T, int CP, bool BACK, bool EXACT>
__global__ void __launch_bounds__(256, CP <= 32 ? (BACK || EXACT || sizeof(T) == 4 ? 2 : 3) : CP <= 64 ? 2 : 1)
    k_query_tile(AttendArgs a) {
  using F = Frag<T>;
  constexpr int NT = kStepLeaves / 8;
  constexpr int STEPS = kStepLeaves / F::STEP;
  constexpr uint32_t SIZE = sizeof(T);
  constexpr bool HELD = SIZE == 2 ? CP <= 64 : CP <= 32 && !BACK;
  constexpr int HOLD = HELD ? CP / F::STEP : 1;
  extern __shared__ __align__(256) char smem[];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Crew crew{tid, int(blockDim.x)};
  const int64_t tile = blockIdx.x;
  const HeadSpan span(a, blockIdx.y);
  const BlockCloud c = a.map.of_tile(tile);
  const bool bias = a.table != nullptr;
  const QueryTileSmem off = query_tile_smem(SIZE, CP, a.kv_cta, a.heads_cta, BACK, bias, a.buckets);
  const uint32_t base = smem_u32(smem);
  uint32_t* s_places = reinterpret_cast<uint32_t*>(smem + off.places);
  int* s_rows = reinterpret_cast<int*>(smem + off.rows);
  uint8_t* s_buckets = reinterpret_cast<uint8_t*>(smem + off.buckets);
  float* s_hist = reinterpret_cast<float*>(smem + off.hist);
  const uint32_t kv_rs = row_bytes<T, CP>(a.kv_cta), q_rs = row_bytes<T, CP>(a.heads_cta);
  const uint32_t stage = kStepLeaves * kv_rs;
  const bool whole = a.width == 16 && a.channels == CP;
  const int columns = span.kvs * CP * int(SIZE) / 16, row_words = a.kv_heads * CP * int(SIZE) / 16;
  const char* k_rows = static_cast<const char*>(a.k) + int64_t(span.kv0) * CP * SIZE;
  const char* v_rows = static_cast<const char*>(a.v) + int64_t(span.kv0) * CP * SIZE;
  const int warps = int(blockDim.x) / 32;

  const int all = a.plan.tile_count[tile];
  const int splits = a.splits;
  const int from = int(int64_t(all) * blockIdx.z / splits);
  const int steps = 2 * (int(int64_t(all) * (blockIdx.z + 1) / splits) - from);
  const uint2* entries = a.plan.entries + tile * a.plan.capacity + from;
  const int points = int(c.n);
  const int64_t* sorted = a.sorted + c.p0;
  const float* leaf_points = a.aabbs + (bias ? leaf_row0(c) * 2 * a.dim : 0);
  const Units units(a.scale);

  auto first_leaf = [&](uint32_t block, int i) { return int(block) * kBlockLeaves + (i & 1) * kStepLeaves; };
  // The warps take turns: one warp asks for the indices (and points) of a step's
  // leaves, one leaf a lane, two steps ahead, and copies its rows one step ahead.
  uint32_t next_index = 0;
  auto fetch = [&](int i) {
    const int leaf = min(first_leaf(entries[i >> 1].x, i) + lane, points - 1);
    next_index = uint32_t(sorted[leaf]);
    if (bias) {
      const float* p = leaf_points + int64_t(leaf) * 2 * a.dim;
      const uint32_t to = base + off.pts + (i % kStages * 3 * kStepLeaves + lane) * 4;
      cp_async<4>(to, p, true);
      cp_async<4>(to + 4 * kStepLeaves, p + 1, true);
      cp_async<4>(to + 8 * kStepLeaves, p + a.dim - 1, a.dim == 3);
    }
  };
  auto copy = [&](int i) {  // by the warp that fetched step i
    const uint32_t at = base + i % kStages * stage;
    copy_words(at + off.k, at + off.v, k_rows, v_rows, checked_row(a, c, next_index) * row_words, columns, kv_rs, lane);
  };
  // Other shapes: the rows go through shared memory to all threads.
  auto publish = [&](int i) { s_places[i % kStages * kStepLeaves + lane] = checked_row(a, c, next_index); };
  auto copy_all = [&](int i) {
    const uint32_t at = base + i % kStages * stage;
    const uint32_t* places = s_places + i % kStages * kStepLeaves;
    auto row_of = [&](int r) { return int(places[r]); };
    const Rows<T, CP> keys{static_cast<const T*>(a.k), a.kv_heads, a.channels, span.kv0, span.kvs, a.width, kv_rs};
    const Rows<T, CP> values{static_cast<const T*>(a.v), a.kv_heads, a.channels, span.kv0, span.kvs, a.width, kv_rs};
    keys.copy(at + off.k, kStepLeaves, row_of, crew);
    values.copy(at + off.v, kStepLeaves, row_of, crew);
  };
  auto sort_pairs = [&](int i, uint32_t mask) {  // distance buckets of step i, for the queries of `mask`
    const int slot = i & 1;
    const BucketTable& table = *reinterpret_cast<const BucketTable*>(smem + off.table);
    uint8_t* to = s_buckets + slot * kTileQueries * kBucketRow;
    const float4* q = reinterpret_cast<const float4*>(smem + off.qpts);
    const float* p = reinterpret_cast<const float*>(smem + off.pts) + i % kStages * 3 * kStepLeaves;
    if (table.crowded) sort_step<true>(to, kBucketRow, table, q, kTileQueries, p, mask);
    else sort_step<false>(to, kBucketRow, table, q, kTileQueries, p, mask);
  };

  clear_padding<T, CP>(smem + off.k, kv_rs, kStages * kStepLeaves, a.kv_cta, a.channels, crew);
  clear_padding<T, CP>(smem + off.v, kv_rs, kStages * kStepLeaves, a.kv_cta, a.channels, crew);
  clear_padding<T, CP>(smem + off.q, q_rs, kTileQueries, a.heads_cta, a.channels, crew);
  if constexpr (BACK) clear_padding<T, CP>(smem + off.d, q_rs, kTileQueries, a.heads_cta, a.channels, crew);
#pragma unroll
  for (int i = 0; i < kStages; ++i)
    if (i < steps && warp == i % warps) {
      fetch(i);
      if (!whole) publish(i);
      else if (i + 1 < kStages) copy(i);
    }
  if (tid < kTileQueries) {
    s_rows[tid] = a.plan.query_row[tile * kTileQueries + tid];
    if (bias) {
      const float* p = a.plan.query_point + tile * 3 * kTileQueries + tid;
      reinterpret_cast<float4*>(smem + off.qpts)[tid] =
          make_float4(-p[0], -p[kTileQueries], -p[2 * kTileQueries], 0.0f);
    }
  }
  if (bias) {
    float* s_bias = reinterpret_cast<float*>(smem + off.bias);
    for (int i = tid; i < span.heads * a.buckets; i += blockDim.x)
      s_bias[(i / a.buckets) * kMaxBuckets + i % a.buckets] = units.of_bias(a.table[int64_t(span.h0) * a.buckets + i]);
    // Rows that a step leaves unsorted are still looked up (and dropped): they must hold offsets.
    for (int i = tid; i < 2 * kTileQueries * kBucketRow / 4; i += blockDim.x)
      reinterpret_cast<uint32_t*>(s_buckets)[i] = 0;
    if constexpr (BACK)
      for (int i = tid; i < a.buckets * int(blockDim.x); i += blockDim.x) s_hist[i] = 0.0f;
  }
  __syncthreads();
  {
    auto row_of = [&](int r) { return s_rows[r]; };
    const Rows<T, CP> q{static_cast<const T*>(a.q), a.heads, a.channels, span.h0, span.heads, a.width, q_rs};
    q.copy(base + off.q, kTileQueries, row_of, crew);
    if constexpr (BACK) {
      const Rows<T, CP> d{static_cast<const T*>(a.grad_out), a.heads, a.channels, span.h0, span.heads, a.width, q_rs};
      d.copy(base + off.d, kTileQueries, row_of, crew);
    }
  }
  if (!whole)
    for (int i = 0; i + 1 < kStages && i < steps; ++i) copy_all(i);
  cp_commit();
  if (bias) reinterpret_cast<BucketTable*>(smem + off.table)->make(a.edges, a.buckets - 1);
  cp_wait<0>();
  __syncthreads();
  if (bias && steps > 0) sort_pairs(0, entries[0].y);

  const int head = warp >> 1, half = warp & 1;
  const bool mine = head < span.heads;
  const int kv = mine ? (span.h0 + head) / a.group - span.kv0 : 0;
  const int g = lane >> 2, t = lane & 3;
  // Byte addresses with the lane's offset; key and value tiles of stage 0.
  const uint32_t q_at = base + off.q + half * 16 * q_rs + head * CP * SIZE + F::lane_a(q_rs, lane);
  const uint32_t d_at = q_at + (off.d - off.q);
  const uint32_t k_at0 = base + off.k + kv * CP * SIZE, v_at0 = base + off.v + kv * CP * SIZE;
  const uint32_t nk = F::lane_nk(kv_rs, lane), kn = F::lane_kn(kv_rs, lane);
  const uint32_t head_bias = base + off.bias + head * kMaxBuckets * 4;
  const uint8_t* near0 = s_buckets + (half * 16 + g) * kBucketRow + 8 * t;
  const uint32_t hist = smem_u32(s_hist + tid);
  const float unit = units.unit;

  typename F::A held_q[HOLD], held_d[BACK ? HOLD : 1];
  if constexpr (HELD) {
    if (mine) hold<T, CP>(held_q, q_at, q_rs);
    if constexpr (BACK)
      if (mine) hold<T, CP>(held_d, d_at, q_rs);
  }
  Pair acc[CP / 8][2] = {};  // rows g and g + 8
  Pair fine[EXACT ? CP / 8 : 1][2] = {};
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};  // forward: running maximum, sum
  float logsum[2] = {INFINITY, INFINITY}, delta[2] = {0.0f, 0.0f};  // backward
  float lift = 1.0f;  // float16: power of two that brings the gradients to order 1
  if constexpr (BACK) {
    lift = gradient_lift<T>(a);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = s_rows[half * 16 + g + 8 * r];
      if (mine && row >= 0) {
        const float2 stats = a.stats_in[int64_t(row) * a.heads + span.h0 + head];
        top[r] = stats.x;
        logsum[r] = stats.y;
        delta[r] = a.delta[int64_t(row) * a.heads + span.h0 + head];
      }
    }
  }

  uint2 entry = steps > 0 ? entries[0] : make_uint2(0, 0), next = entry;
  int copier = (kStages - 1) % warps, fetcher = kStages % warps;  // of steps i + kStages - 1 and i + kStages
  for (int i = 0; i < steps; ++i) {
    cp_wait<kStages - 2>();
    __syncthreads();
    if (i + kStages - 1 < steps) {
      if (!whole) copy_all(i + kStages - 1);
      else if (warp == copier) copy(i + kStages - 1);
      if (warp == fetcher && i + kStages < steps) fetch(i + kStages);
      copier = fetcher;
      if (++fetcher == warps) fetcher = 0;
    }
    if (i + 1 < steps) {
      if (i & 1) next = entries[(i + 1) >> 1];
      if (bias) sort_pairs(i + 1, next.y);
    }
    cp_commit();
    const unsigned mask = entry.y >> (half * 16);
    const int left = points - first_leaf(entry.x, i);
    entry = next;
    const bool fetched = warp == copier && i + kStages < steps;  // (the copier of the next step by now)
    if (!whole && fetched) publish(i + kStages);
    if (!mine || (mask & 0xffffu) == 0 || left <= 0) continue;
    const int slot = i & 1;
    const uint32_t k_at = k_at0 + i % kStages * stage, v_at = v_at0 + i % kStages * stage;
    const uint32_t on[2] = {mask >> g & 1u, mask >> (g + 8) & 1u};
    const uint8_t* near = near0 + slot * kTileQueries * kBucketRow;
    // The step's work: written without branches, so that its chains of dependent
    // instructions overlap; the rare forms (the cloud's last leaves, scales that are
    // not folded) have their own copy.
    auto work = [&](auto biased, auto plain) {
      constexpr bool BIASED = decltype(biased)::value, PLAIN = decltype(plain)::value;
      float s[NT][4];
      logits<T, CP, HELD, BIASED, PLAIN>(s, held_q, q_at, q_rs, k_at + nk, kv_rs, head_bias, near, 8 * kBucketRow,
                                         a.scale * kLog2e, units.folded);
      if constexpr (!PLAIN) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n * 8 + 2 * t + (j & 1) >= left) s[n][j] = -INFINITY;
      }
      if constexpr (!BACK) {
        Pair shrink[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float most = top[r];
#pragma unroll
          for (int n = 0; n < NT; ++n) most = max3(most, s[n][2 * r], s[n][2 * r + 1]);
          most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
          most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
          // Subtracted before the factor, which would round large logits apart.
          const float down = most == -INFINITY ? 0.0f : -most;  // nothing yet: all p are 0
          const float fade = exp2_fast((top[r] + down) * unit);
          Pair add;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 x = unpair(mul2(add2(pair(s[n][2 * r], s[n][2 * r + 1]), both(down)), both(unit)));
            Pair p = pair(exp2_fast(x.x), exp2_fast(x.y));
            add = n == 0 ? p : add2(add, p);
            p = mul2(p, both(F::PEAK_OUT));
            s[n][2 * r] = unpair(p).x;
            s[n][2 * r + 1] = unpair(p).y;
          }
          const float grown = fmaf(sum[r], fade, unpair(add).x + unpair(add).y);
          top[r] = on[r] ? most : top[r];
          sum[r] = on[r] ? grown : sum[r];
          shrink[r] = both(fade);
        }
#pragma unroll
        for (int n0 = 0; n0 < CP / 8; n0 += kChannelGroup) {
          float part[kChannelGroup][4];
          [[maybe_unused]] float low[EXACT ? kChannelGroup : 1][4];
#pragma unroll
          for (int st = 0; st < STEPS; ++st) {
            typename F::A p;
            [[maybe_unused]] typename F::A rest, last;
            from_acc<T>(p, s, st);
            if constexpr (EXACT) rest_of_acc<T>(rest, last, p, s, st);
#pragma unroll
            for (int j = 0; j < kChannelGroup / 2; ++j) {
              typename F::B b;
              F::pair_kn(b, v_at + kn + st * F::STEP * kv_rs + (n0 + 2 * j) * 8 * SIZE, kv_rs);
              if (st == 0) {
                F::mma_first(part[2 * j], p, b[0], b[1]);
                F::mma_first(part[2 * j + 1], p, b[2], b[3]);
                if constexpr (EXACT) {
                  F::mma_first(low[2 * j], rest, b[0], b[1]);
                  F::mma_first(low[2 * j + 1], rest, b[2], b[3]);
                  if constexpr (F::PARTS == 3) {
                    F::mma(low[2 * j], last, b[0], b[1]);
                    F::mma(low[2 * j + 1], last, b[2], b[3]);
                  }
                }
              } else {
                F::mma(part[2 * j], p, b[0], b[1]);
                F::mma(part[2 * j + 1], p, b[2], b[3]);
                if constexpr (EXACT) {
                  F::mma(low[2 * j], rest, b[0], b[1]);
                  F::mma(low[2 * j + 1], rest, b[2], b[3]);
                  if constexpr (F::PARTS == 3) {
                    F::mma(low[2 * j], last, b[0], b[1]);
                    F::mma(low[2 * j + 1], last, b[2], b[3]);
                  }
                }
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            keep_group(acc, n0, r, shrink[r], part, on[r]);
            if constexpr (EXACT) keep_group(fine, n0, r, shrink[r], low, on[r]);
          }
        }
      } else {
        float ds[NT][4];
        multiply_nk<T, CP, NT, HELD, true>(ds, held_d, d_at, q_rs, v_at + nk, kv_rs);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const Pair z = add2(pair(s[n][2 * r], s[n][2 * r + 1]), both(-top[r]));
            const float2 x = unpair(fma2(z, both(unit), both(-logsum[r])));
            Pair p = pair(exp2_fast(x.x), exp2_fast(x.y));
            if constexpr (sizeof(T) == 2) p = mul2(p, both(lift));
            p = mul2(p, add2(pair(ds[n][2 * r], ds[n][2 * r + 1]), both(-delta[r])));
            ds[n][2 * r] = unpair(p).x;
            ds[n][2 * r + 1] = unpair(p).y;
          }
        if constexpr (BIASED) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (on[r]) {
              const uint2 b = *reinterpret_cast<const uint2*>(near + r * 8 * kBucketRow);
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {  // each thread has a column of its own
                  const uint32_t at =
                      hist + __byte_perm(n < 2 ? b.x : b.y, 0, 0x4440 + (n & 1) * 2 + j) * blockDim.x;
                  const float x = lds_f32(at) + ds[n][2 * r + j];
                  asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(x) : "memory");
                }
            }
          }
        }
#pragma unroll
        for (int n0 = 0; n0 < CP / 8; n0 += kChannelGroup) {
          float part[kChannelGroup][4];
#pragma unroll
          for (int st = 0; st < STEPS; ++st) {
            typename F::A p;
            from_acc<T>(p, ds, st);
#pragma unroll
            for (int j = 0; j < kChannelGroup / 2; ++j) {
              typename F::B b;
              F::pair_kn(b, k_at + kn + st * F::STEP * kv_rs + (n0 + 2 * j) * 8 * SIZE, kv_rs);
              if (st == 0) {
                F::mma_first(part[2 * j], p, b[0], b[1]);
                F::mma_first(part[2 * j + 1], p, b[2], b[3]);
              } else {
                F::mma(part[2 * j], p, b[0], b[1]);
                F::mma(part[2 * j + 1], p, b[2], b[3]);
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) keep_group(acc, n0, r, both(1.0f), part, on[r]);
        }
      }
    };
    if (left >= kStepLeaves && units.folded) {
      if (bias) work(std::true_type{}, std::true_type{});
      else work(std::false_type{}, std::true_type{});
    } else {
      if (bias) work(std::true_type{}, std::false_type{});
      else work(std::false_type{}, std::false_type{});
    }
  }

  if (mine) {
    if constexpr (!BACK) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        sum[r] += __shfl_xor_sync(kFullMask, sum[r], 1);
        sum[r] += __shfl_xor_sync(kFullMask, sum[r], 2);
        const int q = half * 16 + g + 8 * r;
        const int row = s_rows[q];
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
            const float2 o = unpair(acc[n][r]);
            part[2 + n * 8 + 2 * t] = o.x;
            part[2 + n * 8 + 2 * t + 1] = o.y;
            if constexpr (EXACT) {
              const float2 f = unpair(fine[n][r]);
              part[2 + CP + n * 8 + 2 * t] = f.x;
              part[2 + CP + n * 8 + 2 * t + 1] = f.y;
            }
          }
          continue;
        }
        if (row < 0) continue;
        const float inv = sum[r] == 0.0f ? 0.0f : 1.0f / F::PEAK_OUT / sum[r];
        T* out = static_cast<T*>(a.out) + (int64_t(row) * a.heads + span.h0 + head) * a.channels;
#pragma unroll
        for (int n = 0; n < CP / 8; ++n)
          store_pair(out, n * 8 + 2 * t, a.channels, unpair(acc[n][r]).x * inv, unpair(acc[n][r]).y * inv, a.wide_out);
        if constexpr (EXACT) {
          float* exact = a.out_exact + (int64_t(row) * a.heads + span.h0 + head) * a.channels;
#pragma unroll
          for (int n = 0; n < CP / 8; ++n)
            store_pair(exact, n * 8 + 2 * t, a.channels, (unpair(acc[n][r]).x + unpair(fine[n][r]).x) * inv,
                       (unpair(acc[n][r]).y + unpair(fine[n][r]).y) * inv, false);
        }
        if (a.stats != nullptr && t == 0) a.stats[int64_t(row) * a.heads + span.h0 + head] = row_stats(top[r], sum[r]);
      }
    } else if (a.grad_q != nullptr) {
      const float back = a.scale / lift;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int q = half * 16 + g + 8 * r, row = s_rows[q];
        if (row < 0) continue;
        if (splits > 1) {
          float* part = a.part + (((int64_t(blockIdx.z) * a.map.num_tiles + tile) * a.heads + span.h0 + head) *
                                      kTileQueries + q) * a.part_row;
#pragma unroll
          for (int n = 0; n < CP / 8; ++n) {
            const float2 x = unpair(acc[n][r]);
            part[n * 8 + 2 * t] = x.x;
            part[n * 8 + 2 * t + 1] = x.y;
          }
          continue;
        }
        T* out = static_cast<T*>(a.grad_q) + (int64_t(row) * a.heads + span.h0 + head) * a.channels;
#pragma unroll
        for (int n = 0; n < CP / 8; ++n)
          store_pair(out, n * 8 + 2 * t, a.channels, unpair(acc[n][r]).x * back, unpair(acc[n][r]).y * back, a.wide_out);
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
        a.table_part[((int64_t(blockIdx.z) * a.map.num_tiles + tile) * a.heads + span.h0) * a.buckets + i] = x / lift;
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
  const dim3 grid(unsigned(a.map.num_tiles), unsigned(head_groups(a)), unsigned(a.splits));
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
