// Building blocks of the block-attention kernels (tbvh_attend_*.cu): matrix
// fragments, shared-memory tiles, row copies and distance buckets.
//
// Products run on warp-level matrix instructions (mma.sync m16n8) with
// accumulators in registers. Every score costs more than its products: mask,
// bucket lookup, bias, exponential, rounding. With 32 channels and a bias the
// forward pass issues 44 thread instructions a selected score (187 M warp instructions
// for 134 M scores), 33 a computed one: a warp computes all 16 rows of a block that any
// of them selected, 1.3 to 1.9 scores for one. The 64 multiply-adds of a score would take
// a tensor-memory instruction a twentieth of that time: issue (58 % of its slots) and the
// waits between a step's barriers bound these kernels, not the matrix pipe (14 % busy).
// And a 16-row instruction lets a warp skip a block that none of its 16 queries selected,
// which a 128-row tile in tensor memory could not.
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

// Pairs of float32 in one 64-bit register: two results an instruction, each
// rounded as the scalar one's.
using Pair = uint64_t;
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ Pair both(float x) { return pair(x, x); }
__device__ __forceinline__ float2 unpair(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// acc[j] = acc[j] * factor + part[j] where `on`, untouched elsewhere.
__device__ __forceinline__ void keep_where(Pair& a0, Pair& a1, Pair& a2, Pair& a3, Pair factor, Pair p0, Pair p1,
                                           Pair p2, Pair p3, uint32_t on) {
  asm("{.reg .pred p;\n setp.ne.u32 p, %9, 0;\n"
      "@p fma.rn.f32x2 %0, %0, %4, %5;\n @p fma.rn.f32x2 %1, %1, %4, %6;\n"
      "@p fma.rn.f32x2 %2, %2, %4, %7;\n @p fma.rn.f32x2 %3, %3, %4, %8;}"
      : "+l"(a0), "+l"(a1), "+l"(a2), "+l"(a3)
      : "l"(factor), "l"(p0), "l"(p1), "l"(p2), "l"(p3), "r"(on));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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

__device__ __forceinline__ float lds_f32(uint32_t addr) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}

// ---- matrix fragments ---------------------------------------------------------------
// Frag<T> multiplies 16 x STEP by STEP x 8 into a float accumulator c[4]: lane
// (g = lane / 4, t = lane % 4) holds rows g and g + 8, columns 2t and 2t + 1.
//
// Operands come from row-major tiles in shared memory, `rs` bytes a row (see
// row_bytes). Each load takes the byte address of its first element plus the
// lane's own offset, which does not change: lane_a / lane_nk / lane_kn.
//  load_a      A from rows of a tile (row = output row, column = depth)
//  pair_nk     B for two neighbouring n-tiles from a tile stored [n][depth]
//  pair_kn     B for two neighbouring n-tiles from a tile stored [depth][n]
//  from_acc    A from an accumulator tile whose columns are the depth
//  mma_first   mma into zeros
// Probabilities enter their products times a power of two, and the sums leave without
// it: PEAK where a row's probabilities sum to 1, PEAK_OUT where the largest of them is 1.
// A sum over the 2,048 keys that a row can have then stays below the type's largest
// value; with 2^-12, what is below 2^-114 of a row's largest may be flushed to zero.
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

  __device__ static __forceinline__ uint32_t lane_a(uint32_t rs, int lane) {
    return ((lane >> 3 & 1) * 8 + (lane & 7)) * rs + (lane >> 4) * 16;
  }
  __device__ static __forceinline__ uint32_t lane_nk(uint32_t rs, int lane) {
    return ((lane >> 4) * 8 + (lane & 7)) * rs + (lane >> 3 & 1) * 16;
  }
  __device__ static __forceinline__ uint32_t lane_kn(uint32_t rs, int lane) { return lane_a(rs, lane); }
  __device__ static __forceinline__ void load_a(A& a, uint32_t at, uint32_t) { ldmatrix4(a.r, at); }
  __device__ static __forceinline__ void pair_nk(B& b, uint32_t at, uint32_t) { ldmatrix4(b, at); }
  __device__ static __forceinline__ void pair_kn(B& b, uint32_t at, uint32_t) { ldmatrix4_t(b, at); }
};

template <>
struct Frag<__nv_bfloat16> : Frag16<__nv_bfloat16> {
  static constexpr int PARTS = 3;  // that hold a float32
  static constexpr float PEAK = 1.0f, PEAK_OUT = 0x1p-12f;
  // Probabilities and their gradients enter the second products in 16 bits: a
  // relative half step of 2^-8 each, the same as the values they multiply.
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
  __device__ static __forceinline__ void mma_first(float (&c)[4], const Frag16<__nv_bfloat16>::A& a, uint32_t b0,
                                                   uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
  __device__ static __forceinline__ float2 unpack(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
  __device__ static __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
  __device__ static __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
};

template <>
struct Frag<__half> : Frag16<__half> {
  static constexpr int PARTS = 2;  // that hold a float32 of [0, 1] to 2^-22 or 2^-25
  // As above with 2^-11 for normal numbers, which begin at 2^-14. A probability of 1 is
  // therefore taken as 2^15, so that it has this relative error down to 2^-29 and 2^-40
  // outright below; dS is scaled by a power of two of its own (gradient_lift): 2^-11
  // relative down to 2^-29 of the most that it can be, 2^-40 of that below.
  static constexpr float PEAK = 0x1p15f, PEAK_OUT = 0x1p15f;
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
  __device__ static __forceinline__ void mma_first(float (&c)[4], const Frag16<__half>::A& a, uint32_t b0,
                                                   uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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
// multiply-add rate. An infinity is a high part of the largest TF32 number and an
// infinite low part, so that the only term with an infinity is its low part times
// the other operand's high part, which has the product's sign (an infinite high part
// would meet low parts of either sign). Times more than 2^11 the term with the other's
// low part may overflow too, to the other side: such a product can be NaN.
template <>
struct Frag<float> {
  static constexpr int STEP = 8;
  static constexpr float PEAK = 1.0f, PEAK_OUT = 0x1p-12f;
  struct A {
    uint32_t hi[4], lo[4];
  };
  using B = float[4];  // two n-tiles

  __device__ static __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.satfinite.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    const float rest = x - __uint_as_float(hi);  // of an infinity, itself; of a NaN, NaN
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
  }
  __device__ static __forceinline__ uint32_t lane_a(uint32_t rs, int lane) {
    return (lane >> 2) * rs + (lane & 3) * 4;
  }
  __device__ static __forceinline__ uint32_t lane_nk(uint32_t rs, int lane) { return lane_a(rs, lane); }
  __device__ static __forceinline__ uint32_t lane_kn(uint32_t rs, int lane) {
    return 2 * (lane & 3) * rs + (lane >> 2) * 4;
  }
  __device__ static __forceinline__ void load_a(A& a, uint32_t at, uint32_t rs) {
    split(lds_f32(at), a.hi[0], a.lo[0]);
    split(lds_f32(at + 8 * rs), a.hi[1], a.lo[1]);
    split(lds_f32(at + 16), a.hi[2], a.lo[2]);
    split(lds_f32(at + 8 * rs + 16), a.hi[3], a.lo[3]);
  }
  __device__ static __forceinline__ void pair_nk(B& b, uint32_t at, uint32_t rs) {
    b[0] = lds_f32(at);
    b[1] = lds_f32(at + 16);
    b[2] = lds_f32(at + 8 * rs);
    b[3] = lds_f32(at + 8 * rs + 16);
  }
  // Depth t of the instruction is row 2t of the tile and depth t + 4 row
  // 2t + 1: the order in which from_acc finds an accumulator's columns.
  __device__ static __forceinline__ void pair_kn(B& b, uint32_t at, uint32_t rs) {
    b[0] = lds_f32(at);
    b[1] = lds_f32(at + rs);
    b[2] = lds_f32(at + 32);
    b[3] = lds_f32(at + rs + 32);
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
  __device__ static __forceinline__ void mma_first(float (&c)[4], const A& a, float b0, float b1) {
    c[0] = c[1] = c[2] = c[3] = 0.0f;
    mma(c, a, b0, b1);
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

// What from_acc's 16-bit rounding leaves of the same elements, as A operands: in one
// part (float16: 2^-22 of them is left), and for bfloat16 in another (2^-24; one part
// would leave 2^-16).
template <typename T, int N>
__device__ __forceinline__ void rest_of_acc(typename Frag<T>::A& rest, typename Frag<T>::A& last,
                                            const typename Frag<T>::A& a, const float (&acc)[N][4], int s) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 near = Frag<T>::unpack(a[i]);
      const float* x = acc[2 * s + (i >> 1)] + 2 * (i & 1);
      const float left[2] = {x[0] - near.x, x[1] - near.y};
      rest[i] = Frag<T>::pack(left[0], left[1]);
      if constexpr (Frag<T>::PARTS == 3) {
        const float2 second = Frag<T>::unpack(rest[i]);
        last[i] = Frag<T>::pack(left[0] - second.x, left[1] - second.y);
      }
    }
  }
}

// ---- tiles in shared memory -----------------------------------------------------------
// Rows past a block's or a list's end repeat its last row: their weights are
// zero, and whoever meets that row's non-finite values has met them already.
//
// [row][head][CP channels], CP the channels rounded up, and 16 bytes of padding
// a row: an odd number of 16-byte words, which puts the eight rows that a
// fragment load touches at once into different banks. A row of whole heads is
// one run of memory in the caller's tensor as well.
template <typename T, int CP>
__host__ __device__ constexpr uint32_t row_bytes(int heads) {
  return uint32_t(heads) * CP * sizeof(T) + 16;
}

// acc[NT][4] += (FRESH: =) A(16 rows) x B^T, B stored [n][channel]. `a` and `b`
// include the lane's offset.
template <typename T, int CP, int NT, bool HELD, bool FRESH>
__device__ __forceinline__ void multiply_nk(float (&acc)[NT][4], const typename Frag<T>::A* held, uint32_t a,
                                            uint32_t a_rs, uint32_t b, uint32_t b_rs) {
#pragma unroll
  for (int s = 0; s < CP / Frag<T>::STEP; ++s) {
    const uint32_t depth = s * Frag<T>::STEP * sizeof(T);
    typename Frag<T>::A fresh;
    if constexpr (!HELD) Frag<T>::load_a(fresh, a + depth, a_rs);
    const typename Frag<T>::A& x = HELD ? held[HELD ? s : 0] : fresh;
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      typename Frag<T>::B y;
      Frag<T>::pair_nk(y, b + j * 16 * b_rs + depth, b_rs);
      if constexpr (sizeof(T) == 4) {
        // The matrix pipe truncates as it adds, all to one side: each depth step is summed by
        // itself and added with rounding.
        float part[2][4];
        Frag<T>::mma_first(part[0], x, y[0], y[1]);
        Frag<T>::mma_first(part[1], x, y[2], y[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[2 * j][i] = FRESH && s == 0 ? part[0][i] : acc[2 * j][i] + part[0][i];
          acc[2 * j + 1][i] = FRESH && s == 0 ? part[1][i] : acc[2 * j + 1][i] + part[1][i];
        }
      } else if (FRESH && s == 0) {
        Frag<T>::mma_first(acc[2 * j], x, y[0], y[1]);
        Frag<T>::mma_first(acc[2 * j + 1], x, y[2], y[3]);
      } else {
        Frag<T>::mma(acc[2 * j], x, y[0], y[1]);
        Frag<T>::mma(acc[2 * j + 1], x, y[2], y[3]);
      }
    }
  }
}

// The fragments of an A operand that stays in registers.
template <typename T, int CP>
__device__ __forceinline__ void hold(typename Frag<T>::A* held, uint32_t a, uint32_t rs) {
#pragma unroll
  for (int s = 0; s < CP / Frag<T>::STEP; ++s) Frag<T>::load_a(held[s], a + s * Frag<T>::STEP * sizeof(T), rs);
}

// Channel tiles are multiplied in groups of this many so that the partial
// products of one group stay in registers.
constexpr int kChannelGroup = 4;

// ---- row copies ------------------------------------------------------------------------
// Widest copy that channels * size and the addresses allow: 16, 8, 4 or 2 bytes.
inline int copy_width(size_t bytes, const void* a, const void* b, const void* c) {
  const uintptr_t all = uintptr_t(a) | uintptr_t(b) | uintptr_t(c) | uintptr_t(bytes);
  for (int w = 16; w > 2; w >>= 1)
    if (all % w == 0) return w;
  return 2;
}

// The threads that share a piece of work, and a thread's number among them.
struct Crew {
  int id, count;
};

// Copies rows of a tensor [row][heads][channels], `here` heads from `first`, into
// a tile; row_of(r) is the packed row number of tile row r,
// negative for zeros. Asynchronous for widths of 4 bytes and more.
template <typename T, int CP>
struct Rows {
  const T* src;
  int heads, channels, first, here, width;
  uint32_t rs;

  template <int BYTES, typename RowOf>
  __device__ __forceinline__ void part(uint32_t dst, int count, RowOf row_of, Crew crew) const {
    constexpr int E = BYTES / int(sizeof(T));
    const int per = channels / E;
    for (int i = crew.id; i < count * per; i += crew.count) {
      const int r = i / per, at = (i - r * per) * E, row = row_of(r);
      const T* p = src + (int64_t(row < 0 ? 0 : row) * heads + first) * channels + at;
      uint32_t d = dst + r * rs + at * uint32_t(sizeof(T));
      for (int h = 0; h < here; ++h, p += channels, d += CP * sizeof(T)) {
        if constexpr (BYTES >= 4) {
          cp_async<BYTES>(d, p, row >= 0);
        } else {
          const uint16_t x = row >= 0 ? *reinterpret_cast<const uint16_t*>(p) : uint16_t(0);
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(d), "h"(x) : "memory");
        }
      }
    }
  }
  template <typename RowOf>
  __device__ __forceinline__ void copy(uint32_t dst, int count, RowOf row_of, Crew crew) const {
    if (width == 16) part<16>(dst, count, row_of, crew);
    else if (width == 8) part<8>(dst, count, row_of, crew);
    else if (width == 4) part<4>(dst, count, row_of, crew);
    else if constexpr (sizeof(T) == 2) part<2>(dst, count, row_of, crew);
  }
};

// 32 rows of two tensors of one shape, copied by ONE warp, where a row's heads are
// one run of `columns` whole 16-byte words on both sides: lane r has row r's place
// in the tensors, in words, and the lanes share the words of the rows.
// The warps of a block take turns, a step each: the same copies spread over all
// warps cost each of them its loop and addresses in every step, three times the
// instructions. (Bulk copies of a row each, issued by one thread one by one,
// took 1.7 times as long a step.)
__device__ __forceinline__ void copy_words(uint32_t a_tile, uint32_t b_tile, const char* a, const char* b,
                                           uint32_t place, int columns, uint32_t rs, int lane) {
  auto put = [](uint32_t dst, const char* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  };
  if (columns <= 32 && (columns & (columns - 1)) == 0) {
    const int rows = 32 / columns, shift = 31 - __clz(columns);  // rows an instruction
    const int column = lane & (columns - 1);
    int r = lane >> shift;
    uint32_t to = r * rs + column * 16;
    const uint32_t step = rows * rs;
    a += column * 16;
    b += column * 16;
#pragma unroll 4
    for (int i = 0; i < columns; ++i, r += rows, to += step) {
      const uint64_t at = uint64_t(__shfl_sync(kFullMask, place, r)) * 16;
      put(a_tile + to, a + at);
      put(b_tile + to, b + at);
    }
  } else {
    int r = lane / columns, column = lane % columns;
    const int dr = 32 / columns, dc = 32 % columns;
    for (int i = 0; i < 32 * columns; i += 32) {
      const uint64_t at = (uint64_t(__shfl_sync(kFullMask, place, r)) + column) * 16;
      const uint32_t to = r * rs + column * 16;
      put(a_tile + to, a + at);
      put(b_tile + to, b + at);
      r += dr;
      column += dc;
      if (column >= columns) {
        column -= columns;
        ++r;
      }
    }
  }
}

// Zeros in the padding channels of tiles, which copies never write.
template <typename T, int CP>
__device__ __forceinline__ void clear_padding(char* tile, uint32_t rs, int rows, int heads, int channels, Crew crew) {
  if (channels == CP) return;
  const int pad = CP - channels;
  for (int i = crew.id; i < rows * heads * pad; i += crew.count) {
    const int at = i % pad, h = i / pad % heads, r = i / (pad * heads);
    *reinterpret_cast<T*>(tile + r * rs + (h * CP + channels + at) * int(sizeof(T))) = T(0.0f);
  }
}

// ---- distance buckets --------------------------------------------------------------------
// bucket(x) = number of edges not above x. A cell holds the floats of one
// exponent and two top mantissa bits: the table has the count at the cell's
// lower end and, where an edge lies inside, that edge, so a lookup is one read
// and one comparison. Only where edges share a cell (closer than 12 to 25 %)
// are they stepped over one by one.
constexpr int kBucketCells = 1024;

struct BucketTable {
  uint2 cell[kBucketCells];  // count * 4, bits of the edge inside (NaN: none)
  float edge[kMaxBuckets];   // ascending; unused and NaN edges at the end as NaN (never counted)
  int crowded;               // some cell holds several edges

  // All threads of the block; a barrier must follow.
  __device__ void make(const float* edges, int count) {
    __shared__ float raw[kMaxBuckets];
    const float nan = __int_as_float(0x7fffffff);
    for (int i = threadIdx.x; i < kMaxBuckets; i += blockDim.x) raw[i] = i < count ? edges[i] : nan;
    if (threadIdx.x == 0) crowded = 0;
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
    for (int i = threadIdx.x; i < kBucketCells; i += blockDim.x) {
      const float low = __uint_as_float(uint32_t(i) << 21);
      int lo = 0, hi = count;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (edge[mid] <= low) lo = mid + 1; else hi = mid;
      }
      // Cells of NaN have low = NaN: no edge counts.
      const float inside = lo < count && __float_as_uint(edge[lo]) >> 21 == uint32_t(i) ? edge[lo] : nan;
      if (lo + 1 < count && __float_as_uint(edge[lo + 1]) >> 21 == uint32_t(i) && low == low) crowded = 1;
      cell[i] = make_uint2(uint32_t(lo) * 4, __float_as_uint(low == low ? inside : nan));
    }
  }
  // Four times the bucket; x >= 0 or NaN (a NaN counts no edge).
  __device__ __forceinline__ uint32_t find4(float x) const {
    const uint2 c = cell[__float_as_uint(x) >> 21];
    uint32_t b = c.x;
    if (x >= __uint_as_float(c.y)) b += 4;
    return b;
  }
  // The same where cells may be crowded.
  __device__ __forceinline__ uint32_t find4_slow(float x) const {
    if (x != x) return 0;
    uint32_t b = cell[__float_as_uint(x) >> 21].x / 4;
    while (b < kMaxBuckets && edge[b] <= x) ++b;
    return b * 4;
  }
  // The bucket of any x.
  __device__ __forceinline__ uint32_t find_any(float x) const {
    if (x > 0.0f) return (crowded ? find4_slow(x) : find4(x)) / 4;
    uint32_t b = 0;
    while (b < kMaxBuckets && edge[b] <= x) ++b;
    return b;
  }
};

// Squared distance of points p (negated) and x, each operation rounded by
// itself, x first. (Not in pairs of float32: the compiler joins their products
// and sums, and distances would miss borders they lie on.) In 2-D z is 0, which
// changes nothing.
__device__ __forceinline__ float pair_distance(float4 minus_p, float x, float y, float z) {
  x = __fadd_rn(x, minus_p.x);
  y = __fadd_rn(y, minus_p.y);
  z = __fadd_rn(z, minus_p.z);
  return __fadd_rn(__fadd_rn(__fmul_rn(x, x), __fmul_rn(y, y)), __fmul_rn(z, z));
}

// Buckets of a step: rows are points p[0..rows), columns the 32 points of `pts`
// ([3][32]). Leaf (or query) n * 8 + 2t + e of a row is byte t * 8 + n * 2 + e,
// so that the eight that lane t of a fragment needs lie side by side; a byte is
// the bucket times four, the offset into a bias row. A thread has four columns
// and every blockDim / 8-th row.
template <bool CROWDED>
__device__ __forceinline__ void sort_step(uint8_t* to, int row_bytes, const BucketTable& table, const float4* p,
                                          int rows, const float* pts, uint32_t wanted) {
  // Four rows a warp and pass; those that no one wants are left out (rows 32 apart share a bit).
  if ((wanted >> (threadIdx.x / 32 * 4 % 32) & 15u) == 0 && blockDim.x >= 256) return;
  const int part = threadIdx.x % 8;  // 2 t + (upper groups)
  const float* c = pts + (part & 1) * 16 + (part >> 1) * 2;
  const float2 x0 = *reinterpret_cast<const float2*>(c), x1 = *reinterpret_cast<const float2*>(c + 8);
  const float2 y0 = *reinterpret_cast<const float2*>(c + 32), y1 = *reinterpret_cast<const float2*>(c + 40);
  const float2 z0 = *reinterpret_cast<const float2*>(c + 64), z1 = *reinterpret_cast<const float2*>(c + 72);
  for (int r = threadIdx.x / 8; r < rows; r += blockDim.x / 8) {
    const float4 q = p[r];
    auto find = [&](float d) { return CROWDED ? table.find4_slow(d) : table.find4(d); };
    const uint32_t b0 = find(pair_distance(q, x0.x, y0.x, z0.x)), b1 = find(pair_distance(q, x0.y, y0.y, z0.y));
    const uint32_t b2 = find(pair_distance(q, x1.x, y1.x, z1.x)), b3 = find(pair_distance(q, x1.y, y1.y, z1.y));
    *reinterpret_cast<uint32_t*>(to + r * row_bytes + part * 4) =
        __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
  }
}

// One score's bias: `row` is the shared address of the head's biases, a multiple
// of 256, so that a byte of buckets put in its place is the bias's address.
__device__ __forceinline__ float bias_of(uint32_t row, uint2 b, int n, int j) {
  return lds_f32(__byte_perm(n < 2 ? b.x : b.y, row, 0x7650 + (n & 1) * 2 + j));
}

// s = logits of 16 rows and 32 columns in units of `unit` (see Units). PLAIN: the
// scale is known to be folded.
template <typename T, int CP, bool HELD, bool BIASED, bool PLAIN>
__device__ __forceinline__ void logits(float (&s)[4][4], const typename Frag<T>::A* held, uint32_t a, uint32_t a_rs,
                                       uint32_t b, uint32_t b_rs, uint32_t bias, const uint8_t* near, int row_step,
                                       float scale, bool folded) {
  if constexpr (BIASED) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint2 w = *reinterpret_cast<const uint2*>(near + r * row_step);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) s[n][2 * r + j] = bias_of(bias, w, n, j);
    }
    if (PLAIN || folded) {
      multiply_nk<T, CP, 4, HELD, false>(s, held, a, a_rs, b, b_rs);
    } else {
      float x[4][4];
      multiply_nk<T, CP, 4, HELD, true>(x, held, a, a_rs, b, b_rs);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = fmaf(x[n][j], scale, s[n][j]);
    }
  } else {
    multiply_nk<T, CP, 4, HELD, true>(s, held, a, a_rs, b, b_rs);
    if (!PLAIN && !folded) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] *= scale;
    }
  }
}

// Logits are kept as z / unit: the bias starts the products' accumulators
// divided by the scale, and scale and base change are one factor in the
// exponential. Scales that this does not suit (negative, tiny, huge) are applied
// to the products instead.
struct Units {
  bool folded;
  float unit, bias;
  // A finite bias stays finite: the type's lowest value everywhere leaves a row its mean.
  __device__ __forceinline__ float of_bias(float x) const {
    const float y = x * bias;
    return fabsf(x) <= FLT_MAX ? fminf(fmaxf(y, -FLT_MAX), FLT_MAX) : y;
  }
  __device__ __forceinline__ explicit Units(float scale) {
    folded = scale >= 0x1p-30f && scale <= 0x1p30f;
    unit = folded ? scale * kLog2e : 1.0f;
    bias = folded ? 1.0f / scale : kLog2e;
  }
};

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
  float2* stats;   // nullable; row_stats of every row and head
  float* out_exact;  // nullable
  int splits;
  float* part;     // splits > 1: [split][tile][head][query] of part_row floats
  int part_row;
  // backward
  const void* grad_out;
  const float2* stats_in;
  float* delta;    // [total_queries][heads] <grad_out, out>
  const unsigned* largest;  // float bits of the largest finite |grad_out| and |value| (float16 only)
  void *grad_q, *grad_k, *grad_v;
  float* table_part;  // [split][tiles][heads][buckets], nullable
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

// Groups of heads_cta query heads.
__host__ __device__ inline int head_groups(const AttendArgs& a) {
  return a.heads_cta >= a.group ? (a.kv_heads + a.kv_cta - 1) / a.kv_cta
                                : a.kv_heads * ((a.group + a.heads_cta - 1) / a.heads_cta);
}

// float16: the power of two that brings the most that |dS| can be, 2 * channels times
// the largest |grad_out| and |value|, to [2^14, 2^15): it stays in float16's range, and
// as many of its small numbers as can be stay normal. Taken out again at the end.
template <typename T>
__device__ __forceinline__ float gradient_lift(const AttendArgs& a) {
  if (a.largest == nullptr) return 1.0f;
  const float most = 2.0f * float(a.channels) * __uint_as_float(a.largest[0]) * __uint_as_float(a.largest[1]);
  return most > 0.0f ? exp2f(14.0f - floorf(log2f(most))) : 1.0f;
}

// What the backward pass keeps of a row's softmax: the largest logit, in units of
// Units, and the base-2 logarithm of the sum (apart, since their sum would round it
// away under large logits). An empty row keeps an infinite sum: its p come out as 0.
__device__ __forceinline__ float2 row_stats(float top, float sum) {
  return sum == 0.0f ? make_float2(0.0f, INFINITY) : make_float2(top, log2f(sum));
}

// Packed row of index `i` of a cloud's order (of its first point, and an error
// bit, where it is none).
__device__ __forceinline__ uint32_t checked_row(const AttendArgs& a, const BlockCloud& c, uint32_t i) {
  if (i >= uint32_t(c.n)) {
    if (a.status) atomicOr(a.status, kDevErrBadIndex);
    i = 0;
  }
  return uint32_t(c.p0) + i;
}

// Packed key row of leaf `leaf` of a cloud, or -1 past its end.
__device__ __forceinline__ int key_row(const AttendArgs& a, const BlockCloud& c, int64_t leaf) {
  if (leaf >= c.n) return -1;
  return int(checked_row(a, c, uint32_t(a.sorted[c.p0 + leaf])));
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
cudaError_t launch_attend_grad_q(const AttendArgs& a, int dtype, cudaStream_t stream);  // joins its splits too
cudaError_t launch_attend_grad_kv(const AttendArgs& a, int dtype, cudaStream_t stream);
// grad_table[values] = sum of part[rows][values] in a fixed order; scratch of kTableRows * values doubles.
cudaError_t launch_table_sum(const float* part, double* scratch, float* grad_table, int64_t rows, int values,
                             cudaStream_t stream);

inline int padded_channels(int channels) { return channels <= 32 ? 32 : channels <= 64 ? 64 : channels <= 96 ? 96 : 128; }

// Raises a kernel's dynamic shared-memory limit where the launch needs it: 48 KB hold the
// kernel's static arrays too. Always to the same size, which leaves them room in an SM's
// 227 KB: with the launch's own, a call in another thread could lower it in between.
constexpr size_t kStaticSmem = 11 * 1024;  // at least those of any kernel this is called for
template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes) {
  return bytes + kStaticSmem > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                                227 * 1024 - int(kStaticSmem))
                                         : cudaSuccess;
}

}  // namespace tbvh
