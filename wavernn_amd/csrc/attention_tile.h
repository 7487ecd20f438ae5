// Shared pieces of the attention kernels (attention_forward.h, attention_backward.h) and of the dense position bias (relative_bias.hip).
//
// Everything is built on one wave tile: 32 "stationary" rows (queries in the forward pass and for dq, keys for dk / dv), one per
// lane column, against 32 "moving" rows.  With v_mfma_f32_32x32x16_bf16 the product  X(moving) * Y(stationary)^T  leaves a lane with
// ONE stationary row and 16 moving rows,
//     moving row of register i = 8 * (i / 4) + 4 * (lane / 32) + i % 4,
// so row statistics of the stationary side are sums inside a lane plus one exchange between the wave's halves, and those 16
// registers are already the right-hand operand of the second product  Z(moving)^T * P : its sum runs over the moving rows, whose
// order is free as long as both operands use the same one.  No score ever goes through shared memory.
//
// float32 goes through the same instructions: a value is the sum of three bfloat16 (8 bits of mantissa each), and a product the six partial
// products that reach 2^-16 of it, added in 32 bits, smallest first.  What is left out is 2^-23 of a product on average and 2^-20 at
// most, the result as exact as the 32-bit matrix instruction's (out at 4096 x 4096 x 128: 8e-7 of the norm, plain float32 products 1.2e-6), and 16 columns of a 32 x 32 tile take
// 6 x 32 cycles where that one takes 8 x 64.
//
// Moving tiles lie in LDS row by row in 16-byte chunks of 8 bfloat16 (three planes for float32).  The first product reads chunk 2c + half of
// a row per lane; the second reads columns with ds_read_b64_tr_b16 (four rows x 16 columns transposed per 16 lanes).
// swizzle() spreads both kinds of read over the banks.
#pragma once
#include <stdint.h>

#include <atomic>

#include "common.h"
#include "../../include/wrnn_mi355.h"

namespace wrnn {
namespace attn {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kLowest = -3.4028235e38f;
constexpr float kFarBias = 2.3e38f, kFarSlope = 0.05f;  // bias_log2
constexpr int kMaxEdges = 128;
constexpr int kMaxDistance = 1024;
constexpr int64_t kMaxRowStride = 1 << 22;

// What the kernels get, by value.  Strides count elements; the last dimension is contiguous.
struct Params {
  const void *q, *k, *v;
  void* out;
  float* lse;    // [B, H, Tq], natural logarithm; -inf where a row has no key
  float* stats;  // [2][B, H, Tq]: a row's reference m (log2 units) and l, the sum of exp2(score - m) over its keys; l = 0 where it has none
  int64_t q_b, q_h, q_t, k_b, k_h, k_t, v_b, v_h, v_t, o_b, o_h, o_t;
  int B, H, Hkv, group, Tq, Tk, D;
  int causal;
  float scale, scale2;      // scale, |scale| * log2(e), above zero
  uint32_t flip;            // sign bit for the stationary operand of the scores where the scale is negative
  const uint8_t* key_mask;  // [B, Tk], non-zero = left out
  int64_t mask_b;
  const int32_t *key_lens, *q_start;
  const float* table;  // [buckets, H]
  int buckets, max_distance, two_sided, exact_side, side, n_edges;
  int edges[kMaxEdges];
  // backward
  const void *dout, *o_in;
  void *dq, *dk, *dv;
  float *delta, *dtable_part;
  int dq_splits, dkv_splits;  // workgroups that share a block of rows, each with part of the other side
  float *dq_part, *dkv_part;  // their sums, where there are several
  int64_t do_b, do_h, do_t, oi_b, oi_h, oi_t, dq_b, dq_h, dq_t, dk_b, dk_h, dk_t, dv_b, dv_h, dv_t;
  int narrow, pack;  // shape of the forward pass
  int splits;        // workgroups that share a block of queries, each with part of the keys
  float* part;
};

// A chunk of 8 elements as the matrix instruction takes it: one bfloat16 plane, or three.
template <class T>
struct Type;
template <>
struct Type<__bf16> {
  static constexpr int NP = 1;
};
template <>
struct Type<float> {
  static constexpr int NP = 3;
};
template <class T>
struct Operand {
  bf16x8 p[Type<T>::NP];
};
template <class T>
struct Raw {  // 8 elements as they come from memory
  typedef T vec __attribute__((ext_vector_type(8)));
  vec x;
  // the values' signs changed where `sign` is the sign bit.  (Here and not in the planes of a float32 operand: there it costs the forward pass 7 %.)
  __device__ __forceinline__ void flip(uint32_t sign) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(__float_as_uint(x[e]) ^ sign);
    } else {
      typedef uint32_t bits __attribute__((ext_vector_type(4)));
      x = __builtin_bit_cast(vec, __builtin_bit_cast(bits, x) ^ (sign | sign >> 16));
    }
  }
};

__device__ __forceinline__ Operand<__bf16> operand(const Raw<__bf16>& r) { return {{r.x}}; }
// One plane of two values, by cutting: the upper half of what the planes before it left (8 bits of mantissa); the subtraction is exact, so
// the three add up to the value itself.
__device__ __forceinline__ uint32_t split2(float& a, float& b, bool more, uint32_t upper = 0xffff0000u, uint32_t uppers = 0x07060302u) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  if (more) {
    a -= __uint_as_float(x & upper);
    b -= __uint_as_float(y & upper);
  }
  return __builtin_amdgcn_perm(y, x, uppers);  // the upper halves of x and y
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void split(f32x8 x, bf16x8 (&p)[3], uint32_t upper = 0xffff0000u, uint32_t uppers = 0x07060302u) {
  u32x4 v[3];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
    for (int n = 0; n < 3; ++n) v[n][j] = split2(a, b, n < 2, upper, uppers);
  }
#pragma unroll
  for (int n = 0; n < 3; ++n) p[n] = __builtin_bit_cast(bf16x8, v[n]);
}
__device__ __forceinline__ Operand<float> operand(const Raw<float>& r) {
  Operand<float> o;
  split(r.x, o.p);
  return o;
}

__device__ __forceinline__ f32x16 mma1(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// One product of 16 columns; between(m) runs after its m-th matrix instruction.
template <class F>
__device__ __forceinline__ f32x16 mma(const Operand<__bf16>& a, const Operand<__bf16>& b, f32x16 c, F&& between) {
  c = mma1(a.p[0], b.p[0], c);
  between(0);
  return c;
}
template <class F>
__device__ __forceinline__ f32x16 mma(const Operand<float>& a, const Operand<float>& b, f32x16 c, F&& between) {
  constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
  for (int m = 0; m < 6; ++m) {
    c = mma1(a.p[pa[m]], b.p[pb[m]], c);
    between(m);
  }
  return c;
}
template <class T>
__device__ __forceinline__ f32x16 mma(const Operand<T>& a, const Operand<T>& b, f32x16 c) {
  return mma(a, b, c, [](int) {});
}

// Two products, instruction by instruction in turn: a product that adds to the one right before it waits for the whole of that one's
// latency.
template <class F>
__device__ __forceinline__ void mma2(const Operand<__bf16>& a0, const Operand<__bf16>& b0, f32x16& c0, const Operand<__bf16>& a1,
                                     const Operand<__bf16>& b1, f32x16& c1, F&& between) {
  c0 = mma1(a0.p[0], b0.p[0], c0);
  between(0);
  c1 = mma1(a1.p[0], b1.p[0], c1);
  between(1);
}
template <class F>
__device__ __forceinline__ void mma2(const Operand<float>& a0, const Operand<float>& b0, f32x16& c0, const Operand<float>& a1,
                                     const Operand<float>& b1, f32x16& c1, F&& between) {
  constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
  for (int m = 0; m < 6; ++m) {
    c0 = mma1(a0.p[pa[m]], b0.p[pb[m]], c0);
    between(2 * m);
    c1 = mma1(a1.p[pa[m]], b1.p[pb[m]], c1);
    between(2 * m + 1);
  }
}

// Work in the matrix instructions' shadow: a 32 x 32 x 16 product keeps the matrix unit for 32 cycles, a vector instruction its unit for 4, and a
// wave issues in order: one that is alone on its SIMD has to have a few vector instructions behind EVERY product, for behind a second
// product they wait with it.  The compiler's scheduler gathers them at the end; shadow<PRODUCTS, PIECES>(m, f) deals f(0) .. f(PIECES - 1)
// out over the products and fences each step.
template <int PRODUCTS, int PIECES, class F>
__device__ __forceinline__ void shadow(int m, F&& f) {
#pragma unroll
  for (int i = m * PIECES / PRODUCTS; i < (m + 1) * PIECES / PRODUCTS; ++i) f(i);
  __builtin_amdgcn_sched_barrier(0);
}

// float32 values on their way to three planes, in steps of one plane of two values (5 vector instructions or 1).
struct Splitter {
  u32x4 w[3];
  float a, b;
  // step i of 12 for 8 values; value(k) gives the k-th
  template <class V>
  __device__ __forceinline__ void step(int i, V&& value) {
    const int j = i / 3, n = i % 3;
    if (n == 0) a = value(2 * j), b = value(2 * j + 1);
    w[n][j] = split2(a, b, n < 2);
  }
  __device__ __forceinline__ Operand<float> get() const {
    return {{__builtin_bit_cast(bf16x8, w[0]), __builtin_bit_cast(bf16x8, w[1]), __builtin_bit_cast(bf16x8, w[2])}};
  }
};

__device__ __forceinline__ int moving_row(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }

// x combined with the other half-wave's: lane l and lane l ^ 32 get the same
__device__ __forceinline__ float both_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Chunk ch (8 elements) of a stationary row of D; what lies past D is zero and not read.  Rows are whole in four elements and start on the bytes of
// four.  Half a chunk at the end of a bfloat16 row: a moving row's is requested as the row's last 16 bytes, so its four elements come second, behind
// four that are in the chunk before, too.  A stationary row has its own in the same place and zeros first, which leaves products over columns right;
// output columns D .. D + 3 then hold what belongs into D - 4 .. D - 1 (column_of).
template <class T>
__device__ __forceinline__ Raw<T> load_chunk(const T* row, int ch, int D) {
  Raw<T> r;
  r.x = {};
  if constexpr (sizeof(T) == 2) {
    typedef __bf16 chunk __attribute__((ext_vector_type(8), aligned(8)));
    if ((D & 4) && ch == D / 8) r.x = __builtin_shufflevector(bf16x4{}, *reinterpret_cast<const bf16x4*>(row + ch * 8), 0, 1, 2, 3, 4, 5, 6, 7);
    else if (ch * 8 < D) r.x = *reinterpret_cast<const chunk*>(row + ch * 8);
  } else {
    f32x4 a = {}, b = {};
    if (ch * 8 < D) a = *reinterpret_cast<const f32x4*>(row + ch * 8);
    if (ch * 8 + 4 < D) b = *reinterpret_cast<const f32x4*>(row + ch * 8 + 4);
    r.x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return r;
}

// The wave's stationary rows: lane column's row in chunks 2c + half.  RAW keeps float32 as it is and splits at every use: half the
// registers of the three planes.
template <class T, int DP, bool RAW>
struct Stationary {
  static constexpr int NC2 = DP / 16;
  Operand<T> o[NC2];
  __device__ __forceinline__ void load(const T* row, int half, int D, bool ok, uint32_t flip = 0) {
#pragma unroll
    for (int c = 0; c < NC2; ++c) {
      Raw<T> r = load_chunk<T>(row, 2 * c + half, D);
      if (!ok) r.x = {};
      r.flip(flip);
      o[c] = operand(r);
    }
  }
  __device__ __forceinline__ const Operand<T>& get(int c) const { return o[c]; }
};
template <class T, int DP>
struct Stationary<T, DP, true> {
  static constexpr int NC2 = DP / 16;
  Raw<T> o[NC2];
  __device__ __forceinline__ void load(const T* row, int half, int D, bool ok, uint32_t flip = 0) {
#pragma unroll
    for (int c = 0; c < NC2; ++c) {
      o[c] = load_chunk<T>(row, 2 * c + half, D);
      if (!ok) o[c].x = {};
      o[c].flip(flip);
    }
  }
  // the constants are hidden from the compiler, or it moves the conversion out of the loop and its results to memory
  __device__ __forceinline__ Operand<T> get(int c) const {
    uint32_t upper = 0xffff0000u, uppers = 0x07060302u;
    asm volatile("" : "+s"(upper), "+s"(uppers));
    Operand<T> x;
    split(o[c].x, x.p, upper, uppers);
    return x;
  }
};

// A tile of ROWS rows of DP elements in LDS, plane after plane.
template <class T, int DP, int ROWS>
struct Tile {
  static constexpr int NP = Type<T>::NP;
  static constexpr int NCH = DP / 8;   // chunks of a row
  static constexpr int ROWB = DP * 2;  // bytes of a row of a plane
  static constexpr int PLANE = ROWS * ROWB, BYTES = NP * PLANE;
  static_assert(ROWB >= 128 && (ROWB & (ROWB - 1)) == 0, "rows of 128 bytes or a power of two more");

  // Chunk position of chunk ch of row r.  Column reads take two neighbouring chunks of four neighbouring rows, row reads one
  // chunk of 32 rows by the first half-wave and its neighbour by the second: pairs of chunks move with the low bits of the row
  // (with rows of 128 bytes, two to a pass over the banks, with the bits above the lowest), the order inside a pair with a higher bit.
  static __device__ __forceinline__ int swizzle(int r, int ch) {
    if (ROWB >= 256) return ch ^ (((r & 7) << 1) | ((r >> 3) & 1));
    return ch ^ ((((r >> 1) & 3) << 1) | ((r >> 3) & 1));
  }
  static __device__ __forceinline__ Operand<T> row_chunk(const char* tile, int r, int ch) {
    Operand<T> o;
#pragma unroll
    for (int n = 0; n < NP; ++n) o.p[n] = *reinterpret_cast<const bf16x8*>(tile + n * PLANE + r * ROWB + swizzle(r, ch) * 16);
    return o;
  }
  static __device__ __forceinline__ void put(char* tile, int r, int ch, const Operand<T>& x) {
#pragma unroll
    for (int n = 0; n < NP; ++n) *reinterpret_cast<bf16x8*>(tile + n * PLANE + r * ROWB + swizzle(r, ch) * 16) = x.p[n];
  }
};

// 16 values of a lane (P or dS) as right-hand operands over 2 x 16 moving rows; split, or rounded to bfloat16, which is what the instruction takes
// beside bfloat16 rows: the sums of so rounded terms (out, dk, dv) are off by 2.2e-3 .. 2.5e-3 of their norm, of which rounding them once at the end is 1.7e-3.
template <class T>
struct Weights {
  Operand<T> o[2];
  __device__ __forceinline__ explicit Weights(const float (&p)[16]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x8 f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = p[8 * s + e];
      if constexpr (sizeof(T) == 2) o[s].p[0] = __builtin_convertvector(f, bf16x8);  // round to nearest even
      else split(f, o[s].p);
    }
  }
};

// The same in bfloat16 as the sum of two operands, 16 bits of mantissa.
struct Weights2 {
  Operand<__bf16> high[2], low[2];
  __device__ __forceinline__ explicit Weights2(const float (&p)[16]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x8 f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = p[8 * s + e];
      high[s].p[0] = __builtin_convertvector(f, bf16x8);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] -= (float)high[s].p[0][e];
      low[s].p[0] = __builtin_convertvector(f, bf16x8);
    }
  }
};

// Left-hand operand X^T of 16 moving rows from row r0 of the tile, output rows d0 .. d0 + 31.  Lane l of a 16-lane group hands in row
// l / 4, columns 4 (l % 4) .. + 3 and gets column l of the four rows.
template <class T, class TL>
__device__ __forceinline__ Operand<T> column_chunk(const char* tile, int r0, int d0, int lane) {
  const int half = lane >> 5, sub = lane & 15, colgrp = (lane >> 4) & 1;
  const int rr = r0 + 4 * half + (sub >> 2), col = d0 + colgrp * 16 + 4 * (sub & 3);
  Operand<T> a;
#pragma unroll
  for (int n = 0; n < TL::NP; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = rr + 8 * u;
      const char* at = tile + n * TL::PLANE + r * TL::ROWB + TL::swizzle(r, col >> 3) * 16 + (col & 7) * 2;
      const bf16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(uintptr_t)(uint32_t)(uintptr_t)at);
#pragma unroll
      for (int e = 0; e < 4; ++e) a.p[n][4 * u + e] = t[e];
    }
  return a;
}

// acc[dt] += X^T W over 32 moving rows from row r0 of the tile, output rows d0 + 32 dt ..
template <class T, class TL, int DT>
__device__ __forceinline__ void column_product(const char* tile, int r0, int d0, const Weights<T>& w, f32x16 (&acc)[DT], int lane) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int s = 0; s < 2; ++s) acc[dt] = mma(column_chunk<T, TL>(tile, r0 + 16 * s, d0 + 32 * dt, lane), w.o[s], acc[dt]);
}

template <class T, class TL, int DT>
__device__ __forceinline__ void column_product(const char* tile, int r0, int d0, const Weights2& w, f32x16 (&acc)[DT], int lane) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const Operand<T> x = column_chunk<T, TL>(tile, r0 + 16 * s, d0 + 32 * dt, lane);
      acc[dt] = mma(x, w.low[s], acc[dt]);
      acc[dt] = mma(x, w.high[s], acc[dt]);
    }
}

// The same for float32 from weights not made yet: value(i) gives weight i of the lane, called once for each in their order.  The first 16
// moving rows' weights are made ahead (or handed in, made in an earlier product's shadow), the others' in the shadow of the first
// products; after(i), AFTER steps of other work, in the shadow of the others.
template <class TL, int DT, int AFTER, class V, class F>
__device__ __forceinline__ void column_product_shadow(const char* tile, int r0, int d0, V&& value, f32x16 (&acc)[DT], int lane, const Splitter* made,
                                                      F&& after) {
  auto chunk = [&](int n) { return column_chunk<float, TL>(tile, r0 + 16 * (n / DT), d0 + 32 * (n % DT), lane); };
  Operand<float> a0 = chunk(0), a1 = chunk(1);
  Splitter first, second;
  if (!made) {
#pragma unroll
    for (int i = 0; i < 12; ++i) first.step(i, value);
  }
  Operand<float> b = made ? made->get() : first.get();
  // Every instruction rounds its sum.  Up to 64 columns the registers have room for the tile's own sums, and the sums over all tiles are rounded
  // once a tile instead of twelve times: at 4096 x 4096 out is off by 3.6e-7 of its norm instead of 7.7e-7, dq, dk and dv by 7.1e-7 instead of
  // 1.0e-6 (a plain float32 product: 1.2e-6), for 0 and 3.5 % of the time.  At 128 columns it would cost the backward pass 17 %.
  constexpr bool OWN = DT == 2;
  f32x16 sum[DT] = {};
  f32x16(&to)[DT] = OWN ? sum : acc;
#pragma unroll
  for (int n = 0; n < 2 * DT; n += 2) {
    if (n == DT) b = second.get();
    Operand<float> n0 = a0, n1 = a1;
    if (n + 2 < 2 * DT) n0 = chunk(n + 2), n1 = chunk(n + 3);
    mma2(a0, b, to[n % DT], a1, b, to[n % DT + 1], [&](int m) {
      if (n < DT) shadow<6 * DT, 12>(6 * n + m, [&](int i) { second.step(i, [&](int k) { return value(8 + k); }); });
      else shadow<6 * DT, AFTER>(6 * (n - DT) + m, after);
    });
    a0 = n0, a1 = n1;
  }
  if constexpr (OWN)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] += sum[dt];
}

// Which rows of a tile of up to 128 may be used, one bit each.
struct RowBits {
  uint64_t lo = 0, hi = 0;
  __device__ __forceinline__ uint32_t of(int sub) const {
    const uint64_t a = lo, b = hi;
    return (uint32_t)((sub & 2 ? b : a) >> (32 * (sub & 1)));
  }
  __device__ __forceinline__ bool at(int r) const {
    const uint64_t a = lo, b = hi;
    return ((r & 64 ? b : a) >> (r & 63)) & 1;
  }
  template <int ROWS>
  __device__ __forceinline__ bool all() const {
    constexpr uint64_t first = ROWS >= 64 ? ~0ull : (1ull << (ROWS & 63)) - 1;
    return (lo & first) == first && (ROWS <= 64 || hi == ~0ull);
  }
};

// The keys of a tile that lengths, reach (end) and mask leave: lane l looks at keys l and l + 64.  The mask's bytes of the tile after are
// requested with each answer.
template <int ROWS>
struct KeyBits {
  const uint8_t* mask;
  int end, lane;
  uint32_t out_lo = 0, out_hi = 0;
  __device__ __forceinline__ KeyBits(const uint8_t* mask_, int end_, int lane_, int first) : mask(mask_), end(end_), lane(lane_) { request(first); }
  __device__ __forceinline__ void request(int key0) {
    if (!mask || end <= 0) return;  // no key at all: nothing to look at (and mask[end - 1] would lie before it)
    out_lo = mask[min(key0 + lane, end - 1)];
    if (ROWS > 64) out_hi = mask[min(key0 + 64 + lane, end - 1)];
  }
  __device__ __forceinline__ RowBits next(int key0) {
    RowBits r;
    r.lo = __ballot(key0 + lane < end && out_lo == 0);
    if (ROWS > 64) r.hi = __ballot(key0 + 64 + lane < end && out_hi == 0);
    request(key0 + ROWS);
    return r;
  }
};

// Rows of a tensor's [.., T, D] slice on their way to an LDS tile: requested a round before they are written to LDS.  Buffer loads check
// every lane against the tile's last byte: rows at or past `limit`, the chunks past D and, by an offset beyond it, rows that a mask leaves out
// come back as zero without a branch.  What lies at keys that are left out (another sequence's values, infinities, NaN) must not reach a
// product, where 0 * NaN would.
template <class T, int DP, int ROWS, int NT>
struct Stage {
  using TL = Tile<T, DP, ROWS>;
  static constexpr int N = ROWS * TL::NCH / NT, STEP = NT / TL::NCH, ES = sizeof(T), PER = 8 * ES / 16;  // PER: 16-byte loads of a chunk
  static_assert(N >= 1 && NT % TL::NCH == 0, "whole rows per pass");
  static constexpr uint32_t kOutside = 0x80000000u;  // past any tile (rows are below 2^22 elements apart)
  Raw<T> r[N];
  const char* base;
  int64_t row_bytes;
  uint32_t off[PER];
  int limit, last;  // rows; bytes of a row that hold data
  __device__ __forceinline__ void start(const T* b, int64_t stride, int rows, int D, int tid) {
    base = reinterpret_cast<const char*>(b);
    row_bytes = stride * ES;
    limit = rows;
    last = D * ES;
    const int ch = tid % TL::NCH, mine = tid / TL::NCH;
    const int back = ES == 2 && (D & 4) && ch == D / 8 ? 8 : 0;  // load_chunk
#pragma unroll
    for (int i = 0; i < PER; ++i)
      off[i] = ch * 8 * ES + 16 * i < last ? (uint32_t)(mine * (int)row_bytes + ch * 8 * ES + 16 * i - back) : kOutside;
  }
  // use: the rows that a mask leaves, or null
  __device__ __forceinline__ void load(int row0, const RowBits* use, int tid) {
    const int rows = min(limit - row0, ROWS);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + (int64_t)row0 * row_bytes), 0,
                                                        rows > 0 ? (rows - 1) * (int)row_bytes + last : 0, 0x00020000);
    if (use && !use->template all<ROWS>()) {
      get(rsrc, [&](int n) { return use->at(tid / TL::NCH + n * STEP) ? 0u : kOutside; });
    } else {
      get(rsrc, [](int) { return 0u; });
    }
  }
  template <class R, class F>
  __device__ __forceinline__ void get(R rsrc, F&& out) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      u32x4 x[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i)
        x[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (off[i] + (uint32_t)(n * STEP * (int)row_bytes)) | out(n), 0, 0);
      if constexpr (PER == 1) r[n].x = __builtin_bit_cast(typename Raw<T>::vec, x[0]);
      else r[n].x = __builtin_shufflevector(__builtin_bit_cast(f32x4, x[0]), __builtin_bit_cast(f32x4, x[1]), 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // the same for rows that are here already
  __device__ __forceinline__ void drop(const RowBits& use, int tid) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (!use.at(tid / TL::NCH + n * STEP)) r[n].x = {};
  }
  __device__ __forceinline__ void store(char* tile, int tid) {
#pragma unroll
    for (int n = 0; n < N; ++n) TL::put(tile, tid / TL::NCH + n * STEP, tid % TL::NCH, operand(r[n]));
  }
  // The same in PIECES steps (float32).
  static constexpr int PIECES = 12 * N;
  __device__ __forceinline__ void store_piece(char* tile, int tid, int i, Splitter& sp) {
    const int n = i / 12;
    sp.step(i % 12, [&](int k) { return r[n].x[k]; });
    if (i % 12 == 11) TL::put(tile, tid / TL::NCH + n * STEP, tid % TL::NCH, sp.get());
  }
};

// The column of a row of D that four output columns from d on belong to, or -1: d itself but for rows that end in half a chunk (load_chunk).
template <class T>
__device__ __forceinline__ int column_of(int d, int D) {
  if (sizeof(T) == 2 && (D & 4) && d >= D - 4) return d == D ? D - 4 : -1;
  return d < D ? d : -1;
}

// A lane's 32 columns x 4 rows of an accumulator as output: column = stationary row, 4 neighbouring d per register group.
template <class T>
__device__ __forceinline__ void store4(T* row, int d, int D, float a, float b, float c, float e) {
  if (d < 0 || d >= D) return;  // D is a whole number of fours
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4*>(row + d) = f32x4{a, b, c, e};
  } else {
    *reinterpret_cast<bf16x4*>(row + d) = bf16x4{(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)e};
  }
}

// Position of row b's query 0 among the keys.  Clamped so that differences of positions stay in 32 bits.
__device__ __forceinline__ int start_of(const Params& p, int b) {
  if (!p.q_start) return p.Tk - p.Tq;
  return min(max(p.q_start[b], -(1 << 29)), 1 << 29);
}

__device__ __forceinline__ int bucket_of(const Params& p, int rel) {
  const int far = p.two_sided ? abs(rel) : max(-rel, 0);
  int n = far;
  if (far >= p.exact_side) {
    n = p.exact_side;
    for (int i = 0; i < p.n_edges; ++i) n += far >= p.edges[i] ? 1 : 0;
  }
  return n + (p.two_sided && rel > 0 ? p.side : 0);
}

// A bias in log2 units.  Past kFarBias in size the change of unit would overflow: from there on it goes with a gentler slope, which keeps
// finite values finite and their order (any two of that size are so far apart that the lower gets no weight), and infinite ones infinite.
__device__ __forceinline__ float bias_log2(float x) {
  const float a = fabsf(x);
  return a <= kFarBias ? x * kLog2e : copysignf(kFarBias * kLog2e + (a - kFarBias) * kFarSlope, x);
}
// The logarithm of a row's sum of exponentials, natural.
__device__ __forceinline__ float row_lse(const Params& p, float m, float l) {
  if (l == 0.f) return -INFINITY;
  const float far = fabsf(m) - kFarBias * kLog2e;
  if (p.table && far > 0.f) return copysignf(fminf(kFarBias + far / kFarSlope, -kLowest), m);
  return (m + log2f(l)) * kLn2;
}

// A row's statistics.  The backward pass works with m and l apart: in the logarithm of their sum, one float, a large m leaves no bit of log2(l) (at
// |m| > 2^24 every key of a row would count whole instead of 1 / l).
__device__ __forceinline__ void store_stats(const Params& p, int64_t row, float m, float l) {
  if (p.lse) p.lse[row] = row_lse(p, m, l);
  if (p.stats) {
    p.stats[row] = m;
    p.stats[(int64_t)p.B * p.H * p.Tq + row] = l;
  }
}
// They as the backward pass takes them: P = exp2(score - m()) * inv().  A row without keys, or none at all: P = exp2(.. - inf) * 0.  Two loads that do
// not wait for each other; the rest where the values are used.
struct RowStats {
  float ref, l;
  __device__ __forceinline__ void load(const Params& p, int64_t row, bool there) {
    ref = l = 0.f;
    if (there) ref = p.stats[row], l = p.stats[(int64_t)p.B * p.H * p.Tq + row];
  }
  __device__ __forceinline__ bool some() const { return l != 0.f; }  // whether the row has a key
  __device__ __forceinline__ float m() const { return l == 0.f ? INFINITY : ref; }
  __device__ __forceinline__ float inv() const { return l == 0.f ? 0.f : 1.f / l; }
};

// The bias of head h by clamped distance, in log2 units: lut[rel + max_distance].
__device__ __forceinline__ void fill_lut(const Params& p, int h, float* lut, int tid, int threads) {
  for (int i = tid; i <= 2 * p.max_distance; i += threads) {
    lut[i] = bias_log2(p.table[(int64_t)bucket_of(p, i - p.max_distance) * p.H + h]);
  }
}

// s = raw products of one 32-key subtile -> scores in log2 units with the bias, or the products as they are; -inf where a pair is left out.
// key0: first key of the subtile; pos: the lane's query position, pos_lo .. pos_hi the wave's; use: bit r = key key0 + r may be used.
template <bool BIAS>
__device__ __forceinline__ void finish_scores(const Params& p, float (&s)[16], int key0, int pos, int pos_lo, int pos_hi, uint32_t use,
                                              const float* lut, int half) {
  if constexpr (BIAS) {
    const int md = p.max_distance;
    if (key0 + 31 - pos_lo <= -md || key0 - pos_hi >= md) {
      const float far = lut[key0 - pos_hi >= md ? 2 * md : 0];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], p.scale2, far);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], p.scale2, lut[min(max(key0 + moving_row(i, half) - pos, -md), md) + md]);
    }
  }
  if (p.causal && key0 + 31 > pos_lo) {
    const int last = pos - key0 - 4 * half;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = moving_row(i, 0) > last ? -INFINITY : s[i];
  }
  if (use != ~0u) {
    const uint32_t mine = use >> (4 * half);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = (mine >> moving_row(i, 0)) & 1 ? s[i] : -INFINITY;
  }
}

// What finish_scores gives, less the row's reference m in log2 units.  Scores without a bias are scaled here, by the one fma that takes m off: no
// rounding in between, the same expression in every kernel (beside a large common level half a step of a score would be as much as the scores
// differ), and an instruction less, which is what the factor 1 / l of P costs in the kernel of dk and dv.
template <bool BIAS>
__device__ __forceinline__ float exponent(const Params& p, float s, float m) {
  return BIAS ? s - m : fmaf(s, p.scale2, -m);
}

// The sum over bucket n's distances of sums[rel + max_distance], in their order.
__device__ __forceinline__ float bucket_sum(const Params& p, const float* sums, int n) {
  const int md = p.max_distance;
  const bool right = p.two_sided && n >= p.side;
  const int m = right ? n - p.side : n, above = m - p.exact_side;
  const int first = above <= 0 ? m : p.edges[above - 1], last = above < 0 ? m + 1 : above < p.n_edges ? p.edges[above] : md + 1;
  float x = 0.f;
  if (right) {
    for (int d = max(first, 1); d < last; ++d) x += sums[md + d];
  } else {
    for (int d = first; d < last; ++d) x += sums[md - d];
    if (!p.two_sided && m == 0)
      for (int d = 1; d <= md; ++d) x += sums[md + d];
  }
  return x;
}

// What a workgroup works on: one of `inner` shares of a tile of a head.  Consecutive items go to one XCD (workgroups are dealt to the eight XCDs in
// turn), so that the tiles of one head share an L2.  Tiles come in the order 0, 1, ..; with `sorted`, where they get shorter in that order
// (causality), an XCD takes tile 0 of all its heads first, then tile 1: the long ones start first and the short ones fill the gaps.
// Launch 8 * ceil(heads * tiles * inner / 8) workgroups.
struct Item {
  int head, tile, share;  // share < 0: nothing to do
  __device__ __forceinline__ Item(int heads, int tiles, int inner, bool sorted) {
    const int x = blockIdx.x & 7, l = blockIdx.x >> 3, n = heads * tiles * inner;
    if (sorted && (heads & 7) == 0) {
      const int per = heads >> 3, u = l / inner;
      share = l - u * inner;
      tile = u / per;
      head = x * per + u - tile * per;
    } else {
      const int per = (n + 7) >> 3, i = x * per + l, u = i / inner;
      share = l < per && i < n ? i - u * inner : -1;
      head = u / tiles;
      tile = u - head * tiles;
    }
  }
};

// One past the last key that some query of row b in [.., last_pos] may use, over lengths, causality and the key mask (a workgroup
// scans the mask's tail once).  `word` is one int of LDS.  All threads of the workgroup call it.
__device__ __forceinline__ int key_end(const Params& p, int b, int last_pos, int* word, int tid, int threads) {
  int end = p.Tk;
  if (p.key_lens) end = min(end, max(p.key_lens[b], 0));
  if (p.causal) end = min(end, max(last_pos + 1, 0));
  if (p.key_mask) {
    const uint8_t* m = p.key_mask + (int64_t)b * p.mask_b;
    for (int hi = end; hi > 0;) {  // blocks of 16 keys a thread from the end, until one holds a key
      const int lo = max(hi - 16 * threads, 0);
      if (tid == 0) *word = 0;
      __syncthreads();
      int last = 0;
      for (int j = lo + tid; j < hi; j += threads)
        if (!m[j]) last = j + 1;
      if (last) atomicMax(word, last);
      __syncthreads();
      const int w = *word;
      __syncthreads();
      if (w) return w;
      hi = lo;
    }
    return 0;
  }
  return end;
}

// ------------------------------------------------------------------ host

constexpr int kLdsBytes = 160 * 1024;

// Lets a kernel have the compute unit's whole LDS, once per kernel and device.
template <class K>
static int allow_lds(K kernel, std::atomic<uint64_t>* done) {
  int dev = 0;
  WRNN_HIP(hipGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (done->load(std::memory_order_acquire) & bit) return 0;
  WRNN_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes));
  done->fetch_or(bit, std::memory_order_release);
  return 0;
}

template <class K>
static int launch(K kernel, std::atomic<uint64_t>* done, int64_t items, int threads, size_t lds, const Params& p, hipStream_t st) {
  if (allow_lds(kernel, done)) return 1;
  WRNN_REQUIRE(lds <= kLdsBytes, "attention: %zu bytes of LDS", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(8 * ((items + 7) / 8))), dim3(threads), lds, st, p);
  WRNN_LAUNCH_CHECK();
  return 0;
}

// Whether every row of a [B, H, T, D] tensor starts on the bytes of four elements.
static inline bool rows_on_four(const void* ptr, int64_t b, int64_t h, int64_t t, int es) {
  return ((reinterpret_cast<uintptr_t>(ptr) | (uintptr_t)(b * es) | (uintptr_t)(h * es) | (uintptr_t)(t * es)) & (4 * es - 1)) == 0;
}

}  // namespace attn

// dtable[n, h] = sum over r of part[r][h][n] (relative_bias.hip).
namespace attn {
template <class T>
int launch_table_sum(const float* part, int rows, int H, int buckets, T* dtable, hipStream_t st);
int bias_params(Params* p, int num_buckets, int max_distance, int bidirectional, const int32_t* edges, const char* who);
}  // namespace attn

// Checks a description and turns it into kernel parameters (attention.hip).
int attention_params(const wrnn_attention_desc* d, attn::Params* p, const char* who);

}  // namespace wrnn
