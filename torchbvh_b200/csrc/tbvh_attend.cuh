// Building blocks of the block-attention kernels (tbvh_attend_*.cu): matrix
// fragments, shared-memory tiles, row copies and distance buckets.
//
// Products run on warp-level matrix instructions (mma.sync m16n8) with
// accumulators in registers. Every score costs more than its products: mask,
// bucket lookup, bias, exponential, rounding. At 32 channels a score is 128
// multiply-adds' worth of flops in the matrix pipe, one exponential (16 a clock
// an SM) and about a dozen other instructions (128 a clock an SM), so the issue
// slots bound these kernels, not the matrix pipe; and a 16-row instruction lets
// a warp skip a block that none of its 16 queries selected, which a 128-row
// tensor-memory tile could not.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tbvh_blocks.h"

namespace tbvh {

constexpr float kLog2e = 1.44269504088896340736f;

// ---- small instructions -----------------------------------------------------------
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool take) {
  const int size = take ? BYTES : 0;  // 0: the destination is filled with zeros, the source not read
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(size)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// ---- matrix fragments ---------------------------------------------------------------
// Frag<T> multiplies 16 x STEP by STEP x 8 into a float accumulator c[4]: lane
// (g = lane / 4, t = lane % 4) holds rows g and g + 8, columns 2t and 2t + 1.
//
// Tiles in shared memory are row-major with LD elements a row (see Tile).
//  load_a      A from rows of a tile (row = output row, column = depth)
//  pair_nk     B for two neighbouring n-tiles from a tile stored [n][depth]
//  pair_kn     B for two neighbouring n-tiles from a tile stored [depth][n]
//  from_acc    A from an accumulator tile whose columns are the depth
template <typename T>
struct Frag;

template <typename T>
struct Frag16 {
  static constexpr int STEP = 16;
  struct A {
    uint32_t r[4];
    __device__ __forceinline__ uint32_t& operator[](int i) { return r[i]; }
    __device__ __forceinline__ uint32_t operator[](int i) const { return r[i]; }
  };
  using B = uint32_t[4];  // two n-tiles

  __device__ static __forceinline__ void load_a(A& a, const T* tile, int ld, int row, int k, int lane) {
    const int m = lane >> 3, r = lane & 7;
    ldmatrix4(a.r, smem_u32(tile + (row + (m & 1) * 8 + r) * ld + k + (m >> 1) * 8));
  }
  __device__ static __forceinline__ void pair_nk(B& b, const T* tile, int ld, int n, int k, int lane) {
    const int m = lane >> 3, r = lane & 7;
    ldmatrix4(b, smem_u32(tile + (n + (m >> 1) * 8 + r) * ld + k + (m & 1) * 8));
  }
  __device__ static __forceinline__ void pair_kn(B& b, const T* tile, int ld, int k, int n, int lane) {
    const int m = lane >> 3, r = lane & 7;
    ldmatrix4_t(b, smem_u32(tile + (k + (m & 1) * 8 + r) * ld + n + (m >> 1) * 8));
  }
};

template <>
struct Frag<__nv_bfloat16> : Frag16<__nv_bfloat16> {
  // Probabilities and their gradients enter the second products in 16 bits: a
  // relative half step of 2^-9 each, the same as the values they multiply.
  __device__ static __forceinline__ uint32_t pack(float x, float y) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
  }
  __device__ static __forceinline__ void mma(float (&c)[4], const Frag16<__nv_bfloat16>::A& a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static __forceinline__ float2 unpack(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
  __device__ static __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
  __device__ static __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
};

template <>
struct Frag<__half> : Frag16<__half> {
  // As above with 2^-12; the backward pass scales by a power of two so that
  // small gradients stay normal numbers.
  __device__ static __forceinline__ uint32_t pack(float x, float y) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
  }
  __device__ static __forceinline__ void mma(float (&c)[4], const Frag16<__half>::A& a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static __forceinline__ float2 unpack(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
  __device__ static __forceinline__ float to_float(__half x) { return __half2float(x); }
  __device__ static __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
};

// float32 features: each operand is split into two TF32 numbers (11 + 11 bits)
// and the product taken as hi hi + hi lo + lo hi; what is dropped is 2^-22 of
// it. Three TF32 products cost six bf16 ones and still twice the plain
// multiply-add rate.
template <>
struct Frag<float> {
  static constexpr int STEP = 8;
  struct A {
    uint32_t hi[4], lo[4];
  };
  using B = float[4];  // two n-tiles

  __device__ static __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    const float rest = x - __uint_as_float(hi);
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
    // An infinity or NaN is carried by the high part alone.
    if (!(fabsf(x) <= FLT_MAX)) lo = 0;
  }
  __device__ static __forceinline__ void load_a(A& a, const float* tile, int ld, int row, int k, int lane) {
    const float* p = tile + (row + (lane >> 2)) * ld + k + (lane & 3);
    split(p[0], a.hi[0], a.lo[0]);
    split(p[8 * ld], a.hi[1], a.lo[1]);
    split(p[4], a.hi[2], a.lo[2]);
    split(p[8 * ld + 4], a.hi[3], a.lo[3]);
  }
  __device__ static __forceinline__ void pair_nk(B& b, const float* tile, int ld, int n, int k, int lane) {
    const float* p = tile + (n + (lane >> 2)) * ld + k + (lane & 3);
    b[0] = p[0];
    b[1] = p[4];
    b[2] = p[8 * ld];
    b[3] = p[8 * ld + 4];
  }
  // Depth t of the instruction is row 2t of the tile and depth t + 4 row
  // 2t + 1: the order in which from_acc finds an accumulator's columns.
  __device__ static __forceinline__ void pair_kn(B& b, const float* tile, int ld, int k, int n, int lane) {
    const float* p = tile + (k + 2 * (lane & 3)) * ld + n + (lane >> 2);
    b[0] = p[0];
    b[1] = p[ld];
    b[2] = p[8];
    b[3] = p[ld + 8];
  }
  __device__ static __forceinline__ void mma1(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static __forceinline__ void mma(float (&c)[4], const A& a, float b0, float b1) {
    uint32_t h0, l0, h1, l1;
    split(b0, h0, l0);
    split(b1, h1, l1);
    mma1(c, a.lo, h0, h1);
    mma1(c, a.hi, l0, l1);
    mma1(c, a.hi, h0, h1);
  }
  __device__ static __forceinline__ float to_float(float x) { return x; }
  __device__ static __forceinline__ float from_float(float x) { return x; }
};

// A operand of depth step `s` from accumulator tiles acc[..][4] whose columns
// are the depth (16-bit: two tiles a step, TF32: one).
template <typename T, int N>
__device__ __forceinline__ void from_acc(typename Frag<T>::A& a, const float (&acc)[N][4], int s) {
  if constexpr (sizeof(T) == 2) {
    a[0] = Frag<T>::pack(acc[2 * s][0], acc[2 * s][1]);
    a[1] = Frag<T>::pack(acc[2 * s][2], acc[2 * s][3]);
    a[2] = Frag<T>::pack(acc[2 * s + 1][0], acc[2 * s + 1][1]);
    a[3] = Frag<T>::pack(acc[2 * s + 1][2], acc[2 * s + 1][3]);
  } else {
    Frag<T>::split(acc[s][0], a.hi[0], a.lo[0]);
    Frag<T>::split(acc[s][2], a.hi[1], a.lo[1]);
    Frag<T>::split(acc[s][1], a.hi[2], a.lo[2]);
    Frag<T>::split(acc[s][3], a.hi[3], a.lo[3]);
  }
}

// What from_acc's 16-bit rounding leaves of the same elements, as an A operand.
template <typename T, int N>
__device__ __forceinline__ void rest_of_acc(typename Frag<T>::A& rest, const typename Frag<T>::A& a,
                                            const float (&acc)[N][4], int s) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 near = Frag<T>::unpack(a[i]);
      const float* x = acc[2 * s + (i >> 1)] + 2 * (i & 1);
      rest[i] = Frag<T>::pack(x[0] - near.x, x[1] - near.y);
    }
  }
}

// ---- tiles in shared memory -----------------------------------------------------------
// Rows of CP elements (the channels rounded up) and 16 bytes of padding, which
// puts the eight rows that a fragment load touches at once into different banks.
template <typename T, int CP>
struct Tile {
  static constexpr int LD = CP + 16 / int(sizeof(T));
  __host__ __device__ static constexpr int elems(int rows) { return rows * LD; }
};

// acc[NT][4] += A(16 rows of `a_tile` from `row`) x B^T, B stored [n][channel], n from n0.
template <typename T, int CP, int NT, bool HELD>
__device__ __forceinline__ void multiply_nk(float (&acc)[NT][4], const typename Frag<T>::A* held, const T* a_tile,
                                            int row, const T* b_tile, int n0, int lane) {
  constexpr int LD = Tile<T, CP>::LD;
#pragma unroll
  for (int s = 0; s < CP / Frag<T>::STEP; ++s) {
    typename Frag<T>::A fresh;
    if constexpr (!HELD) Frag<T>::load_a(fresh, a_tile, LD, row, s * Frag<T>::STEP, lane);
    const typename Frag<T>::A& a = HELD ? held[HELD ? s : 0] : fresh;
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      typename Frag<T>::B b;
      Frag<T>::pair_nk(b, b_tile, LD, n0 + j * 16, s * Frag<T>::STEP, lane);
      Frag<T>::mma(acc[2 * j], a, b[0], b[1]);
      Frag<T>::mma(acc[2 * j + 1], a, b[2], b[3]);
    }
  }
}

// The fragments of an A operand that stays in registers.
template <typename T, int CP>
__device__ __forceinline__ void hold(typename Frag<T>::A* held, const T* a_tile, int row, int lane) {
#pragma unroll
  for (int s = 0; s < CP / Frag<T>::STEP; ++s)
    Frag<T>::load_a(held[s], a_tile, Tile<T, CP>::LD, row, s * Frag<T>::STEP, lane);
}

// Channel tiles are multiplied in groups of this many so that the partial
// products of one group stay in registers.
constexpr int kChannelGroup = 4;

// ---- row copies ------------------------------------------------------------------------
// Widest copy that channels * size and the addresses allow: 16, 8, 4 or 2 bytes.
inline int copy_width(size_t row_bytes, const void* a, const void* b, const void* c) {
  const uintptr_t all = uintptr_t(a) | uintptr_t(b) | uintptr_t(c) | uintptr_t(row_bytes);
  for (int w = 16; w > 2; w >>= 1)
    if (all % w == 0) return w;
  return 2;
}

// Copies rows rows[0..count) (packed row numbers, negative: zeros) of a tensor
// [row][heads][channels] into tiles dst[head][row][LD], heads_here heads from
// `first`, `step` apart. Asynchronous for widths of 4 bytes and more.
template <typename T, int CP, int BYTES>
__device__ __forceinline__ void copy_rows_w(T* dst, int tile_elems, const T* src, const int* rows, int count,
                                            int heads, int channels, int first, int heads_here, int head_step) {
  constexpr int E = BYTES / int(sizeof(T));
  constexpr int LD = Tile<T, CP>::LD;
  const bool full = channels == CP;
  const int per = full ? CP / E : channels / E;
  for (int i = threadIdx.x; i < count * per; i += blockDim.x) {
    const int r = full ? i / (CP / E) : i / per;
    const int at = (i - r * per) * E;
    const int row = rows[r];
    const T* p = src + (int64_t(row < 0 ? 0 : row) * heads + first) * channels + at;
    T* d = dst + r * LD + at;
    for (int h = 0; h < heads_here; ++h, p += int64_t(head_step) * channels, d += tile_elems) {
      if constexpr (BYTES >= 4) cp_async<BYTES>(smem_u32(d), p, row >= 0);
      else *d = row >= 0 ? *p : T(0.0f);
    }
  }
}

template <typename T, int CP>
__device__ __forceinline__ void copy_rows(T* dst, int tile_elems, const T* src, const int* rows, int count, int heads,
                                          int channels, int first, int heads_here, int width, int step = 1) {
  if (width == 16) copy_rows_w<T, CP, 16>(dst, tile_elems, src, rows, count, heads, channels, first, heads_here, step);
  else if (width == 8) copy_rows_w<T, CP, 8>(dst, tile_elems, src, rows, count, heads, channels, first, heads_here, step);
  else if (width == 4) copy_rows_w<T, CP, 4>(dst, tile_elems, src, rows, count, heads, channels, first, heads_here, step);
  else if constexpr (sizeof(T) == 2)
    copy_rows_w<T, CP, 2>(dst, tile_elems, src, rows, count, heads, channels, first, heads_here, step);
}

// Zeros in the padding channels of tiles that copies never write.
template <typename T, int CP>
__device__ __forceinline__ void clear_padding(T* tiles, int rows, int channels) {
  if (channels == CP) return;
  constexpr int LD = Tile<T, CP>::LD;
  const int pad = CP - channels;
  for (int i = threadIdx.x; i < rows * pad; i += blockDim.x) tiles[(i / pad) * LD + channels + i % pad] = T(0.0f);
}

// ---- distance buckets --------------------------------------------------------------------
// bucket(x) = number of edges not above x. A cell holds the floats of one
// exponent and three top mantissa bits, counted from the smallest positive edge:
// 511 cells reach 2^63 times that edge, one takes all that is larger. A cell's
// entry is the count at its lower end and, where one edge lies inside, that
// edge: a lookup is one read and one comparison. Only where edges are closer
// than a cell (12 %) are they stepped over one by one.
constexpr int kBucketCells = 512;

struct BucketTable {
  float edge[kMaxBuckets];  // ascending; unused and NaN edges at the end as NaN (never counted)
  uint2 cell[kBucketCells]; // count | crowded << 8, bits of the edge inside (NaN: none)
  int first;                // cell number of cell[0]
  int not_positive;         // edges that are zero or negative

  // All threads of the block; a barrier must follow.
  __device__ void make(const float* edges, int count) {
    __shared__ float raw[kMaxBuckets];
    const float nan = __int_as_float(0x7fffffff);
    for (int i = threadIdx.x; i < kMaxBuckets; i += blockDim.x) raw[i] = i < count ? edges[i] : nan;
    __syncthreads();
    for (int i = threadIdx.x; i < kMaxBuckets; i += blockDim.x) {
      const float x = raw[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) {
        const float y = raw[j];
        rank += y != y ? x != x && j < i : x != x || y < x || (y == x && j < i);
      }
      if (i >= count) rank = i;  // behind every edge
      edge[rank] = x;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int n = 0;
      while (n < count && edge[n] <= 0.0f) ++n;
      not_positive = n;
      first = n < count && edge[n] == edge[n] ? int(__float_as_uint(edge[n]) >> 20) - 1 : 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBucketCells; i += blockDim.x) {
      const int n = max(first + i, 0);
      // Edges up to the cell's lower end; cell 0 starts at 0.
      const float low = i == 0 ? 0.0f : __uint_as_float(uint32_t(n) << 20);
      const float high = i + 1 == kBucketCells ? INFINITY : __uint_as_float(uint32_t(n + 1) << 20);
      int lo = 0, hi = count;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (edge[mid] <= low) lo = mid + 1; else hi = mid;
      }
      int inside = 0;
      while (inside < 2 && lo + inside < count && (edge[lo + inside] < high || i + 1 == kBucketCells) &&
             edge[lo + inside] == edge[lo + inside])
        ++inside;
      cell[i] = make_uint2(uint32_t(lo) | (inside > 1 ? 256u : 0u),
                           __float_as_uint(inside > 0 ? edge[lo] : nan));
    }
  }
  // x >= 0 or NaN (a NaN counts no edge).
  __device__ __forceinline__ int find(float x) const {
    const int i = min(max(int(__float_as_uint(x) >> 20) - first, 0), kBucketCells - 1);
    const uint2 c = cell[i];
    int b = int(c.x) + (x >= __uint_as_float(c.y) ? 1 : 0);
    if (b >= 256) {  // several edges in the cell
      b = int(c.x) - 256;
      while (b < kMaxBuckets && edge[b] <= x) ++b;
    }
    return x == x ? b : 0;
  }
  // Any x.
  __device__ __forceinline__ int find_any(float x) const {
    if (x > 0.0f) return find(x);
    int b = 0;
    while (b < kMaxBuckets && edge[b] <= x) ++b;
    return b;
  }
};

// Squared distance of a pair, each operation rounded.
__device__ __forceinline__ float pair_distance(float qx, float qy, float qz, float px, float py, float pz, bool three) {
  const float x = __fsub_rn(qx, px), y = __fsub_rn(qy, py);
  float d = __fadd_rn(__fmul_rn(x, x), __fmul_rn(y, y));
  if (three) {
    const float z = __fsub_rn(qz, pz);
    d = __fadd_rn(d, __fmul_rn(z, z));
  }
  return d;
}

// ---- arguments shared by the kernels --------------------------------------------------------
struct AttendArgs {
  BlockMap map;
  BlockPlan plan;
  const float* aabbs;
  const int64_t* sorted;
  int dim;
  const void *q, *k, *v;
  int heads, kv_heads, channels;
  int group;       // query heads per key/value head
  int heads_cta;   // query heads of one thread block
  int kv_cta;      // key/value heads of one thread block
  float scale;     // natural
  const float* table;  // nullable: no bias
  const float* edges;
  int buckets;
  int width;       // bytes of one row copy
  bool wide_out;   // pairs of 16-bit outputs are 4-byte aligned
  unsigned* status;
  // forward
  void* out;
  float* lse;      // nullable
  float* out_exact;  // nullable
  int splits;
  float* part;     // splits > 1: [split][tile][head][query] of part_row floats
  int part_row;
  // backward
  const void* grad_out;
  const float* lse_in;
  float* delta;    // [total_queries][heads] <grad_out, out>
  const unsigned* grad_max;  // float bits of the largest |grad_out| (float16 only)
  void *grad_q, *grad_k, *grad_v;
  float* table_part;  // [tiles][heads][buckets], nullable
};

// First query head, count, first key/value head and count of blockIdx.y.
struct HeadSpan {
  int h0, heads, kv0, kvs;
  __device__ __forceinline__ explicit HeadSpan(const AttendArgs& a, int y) {
    if (a.heads_cta >= a.group) {  // whole groups
      kv0 = y * a.kv_cta;
      kvs = min(a.kv_cta, a.kv_heads - kv0);
      h0 = kv0 * a.group;
      heads = kvs * a.group;
    } else {  // part of one group
      const int parts = (a.group + a.heads_cta - 1) / a.heads_cta;
      kv0 = y / parts;
      kvs = 1;
      const int from = (y % parts) * a.heads_cta;
      h0 = kv0 * a.group + from;
      heads = min(a.heads_cta, a.group - from);
    }
  }
};

// float16: the power of two that brings the largest |grad_out| to [1, 2), so that
// products of small gradients stay normal numbers; taken out again at the end.
template <typename T>
__device__ __forceinline__ float gradient_lift(const AttendArgs& a) {
  if (a.grad_max == nullptr) return 1.0f;
  const float most = __uint_as_float(*a.grad_max);
  if (!(most > 0.0f && most <= FLT_MAX)) return 1.0f;
  return exp2f(-floorf(log2f(most)));
}

// Packed key row of leaf `leaf` of a cloud, or -1 past its end.
__device__ __forceinline__ int key_row(const AttendArgs& a, const BlockCloud& c, int64_t leaf) {
  if (leaf >= c.n) return -1;
  const int64_t i = a.sorted[c.p0 + leaf];
  if (uint64_t(i) >= uint64_t(c.n)) {
    if (a.status) atomicOr(a.status, kDevErrBadIndex);
    return -1;
  }
  return int(c.p0 + i);
}

// First leaf row of a cloud's node rows.
__device__ __forceinline__ int64_t leaf_row0(const BlockCloud& c) {
  const int level = ceil_log2_i64(c.n);
  return c.row0 + level_row_offset(c.n, level, level);
}

// Stores two neighbouring channels of a row, those that exist.
template <typename T>
__device__ __forceinline__ void store_pair(T* row, int at, int channels, float x, float y, bool wide) {
  if constexpr (sizeof(T) == 2) {
    if (wide && at + 1 < channels) {
      *reinterpret_cast<uint32_t*>(row + at) = Frag<T>::pack(x, y);
      return;
    }
  }
  if (at < channels) row[at] = Frag<T>::from_float(x);
  if (at + 1 < channels) row[at + 1] = Frag<T>::from_float(y);
}

// Partial rows of launch_table_sum's scratch (64-bit values each).
constexpr int kTableRows = 64;

// ---- host ----------------------------------------------------------------------------------
cudaError_t launch_attend_forward(const AttendArgs& a, int dtype, cudaStream_t stream);
cudaError_t launch_attend_forward_exact(const AttendArgs& a, int dtype, cudaStream_t stream);
cudaError_t launch_attend_merge(const AttendArgs& a, int dtype, cudaStream_t stream);
cudaError_t launch_attend_grad_q(const AttendArgs& a, int dtype, cudaStream_t stream);
cudaError_t launch_attend_grad_kv(const AttendArgs& a, int dtype, cudaStream_t stream);
// grad_table[values] = sum of part[rows][values] in a fixed order; scratch of kTableRows * values doubles.
cudaError_t launch_table_sum(const float* part, double* scratch, float* grad_table, int64_t rows, int values,
                             cudaStream_t stream);

inline int padded_channels(int channels) { return channels <= 32 ? 32 : channels <= 64 ? 64 : channels <= 96 ? 96 : 128; }

// Raises a kernel's dynamic shared-memory limit, once per device and kernel.
template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes) {
  return bytes > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes))
                           : cudaSuccess;
}

}  // namespace tbvh
