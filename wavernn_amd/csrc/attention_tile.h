// Shared device pieces of the attention kernels (attention.hip, attention_backward.hip).
//
// Everything is built on one wave tile: 32 "stationary" rows (queries in the forward pass and for dq, keys for dk / dv), one per
// lane column, against 32 "moving" rows.  With v_mfma_f32_32x32x* the product  X(moving) * Y(stationary)^T  leaves a lane with ONE
// stationary row and 16 moving rows,
//     moving row of register i = 8 * (i / 4) + 4 * (lane / 32) + i % 4,
// so row statistics of the stationary side are sums inside a lane plus one exchange between the wave's halves, and those 16
// registers are already the right-hand operand of the second product  Z(moving)^T * P : its sum runs over the moving rows, whose
// order is free as long as both operands use the same one.  No score ever goes through shared memory.
//
// Moving tiles lie in LDS row by row in 16-byte chunks.  The first product reads chunk 2c + half of a row per lane; the second
// reads columns: bfloat16 with ds_read_b64_tr_b16 (four rows x 16 columns transposed per 16 lanes), float32 one word per lane.
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

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxEdges = 128;
constexpr int kMaxDistance = 1024;

// What the kernels get, by value.  Strides count elements; the last dimension is contiguous.
struct Params {
  const void *q, *k, *v;
  void* out;
  float* lse;  // [B, H, Tq], natural logarithm; -inf where a row has no key
  int64_t q_b, q_h, q_t, k_b, k_h, k_t, v_b, v_h, v_t, o_b, o_h, o_t;
  int B, H, Hkv, group, Tq, Tk, D;
  int causal, vec;          // vec: every row of every tensor starts on 16 bytes and D fills whole chunks
  float scale, scale2;      // scale, scale * log2(e)
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
  int64_t do_b, do_h, do_t, oi_b, oi_h, oi_t, dq_b, dq_h, dq_t, dk_b, dk_h, dk_t, dv_b, dv_h, dv_t;
  // keys split over workgroups (few queries)
  int splits, pack;
  float* part;
};

template <class T>
struct Type;
template <>
struct Type<__bf16> {
  using chunk = bf16x8;
  static constexpr int CE = 8;  // elements of a 16-byte chunk
  static __device__ __forceinline__ f32x16 mma(chunk a, chunk b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Type<float> {
  using chunk = f32x4;
  static constexpr int CE = 4;
  // element e of the two halves' chunks makes one K = 2 product
  static __device__ __forceinline__ f32x16 mma(chunk a, chunk b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ int moving_row(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }

// the other half-wave's value
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

template <class T>
__device__ __forceinline__ typename Type<T>::chunk load_chunk(const T* row, int ch, int D, bool vec) {
  using chunk = typename Type<T>::chunk;
  constexpr int CE = Type<T>::CE;
  chunk r = {};
  if (vec) {
    if (ch * CE < D) r = *reinterpret_cast<const chunk*>(row + ch * CE);
  } else {
#pragma unroll
    for (int e = 0; e < CE; ++e)
      if (ch * CE + e < D) r[e] = row[ch * CE + e];
  }
  return r;
}

// A tile of ROWS rows of DP elements in LDS.
template <class T, int DP>
struct Tile {
  using chunk = typename Type<T>::chunk;
  static constexpr int CE = Type<T>::CE;
  static constexpr int NCH = DP / CE;       // chunks of a row
  static constexpr int ROWB = DP * sizeof(T);
  static_assert(ROWB >= 128 && (ROWB & (ROWB - 1)) == 0, "rows of 128 bytes or a power of two more");

  // Chunk position of chunk ch of row r.  Column reads take two neighbouring chunks of four neighbouring rows, row reads one
  // chunk of 32 rows by the first half-wave and its neighbour by the second: pairs of chunks move with the low bits of the row
  // (with rows of 128 bytes, two to a pass over the banks, with the bits above the lowest), the order inside a pair with a higher bit.
  static __device__ __forceinline__ int swizzle(int r, int ch) {
    if (ROWB >= 256) return ch ^ (((r & 7) << 1) | ((r >> 3) & 1));
    return ch ^ ((((r >> 1) & 3) << 1) | ((r >> 3) & 1));
  }
  static __device__ __forceinline__ chunk row_chunk(const char* tile, int r, int ch) {
    return *reinterpret_cast<const chunk*>(tile + r * ROWB + swizzle(r, ch) * 16);
  }
  static __device__ __forceinline__ void put(char* tile, int r, int ch, chunk x) {
    *reinterpret_cast<chunk*>(tile + r * ROWB + swizzle(r, ch) * 16) = x;
  }
};

// acc[dt] += X^T P over 32 moving rows from `r0` of the tile; p holds a lane's 16 values in register order.
template <class T, int DP, int DT>
struct ColumnProduct;
template <int DP, int DT>
struct ColumnProduct<__bf16, DP, DT> {
  static __device__ __forceinline__ void run(const char* tile, int r0, int d0, const float (&p)[16], f32x16 (&acc)[DT], int lane) {
    using TL = Tile<__bf16, DP>;
    bf16x8 b[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x8 f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = p[8 * s + e];
      b[s] = __builtin_convertvector(f, bf16x8);  // round to nearest even
    }
    // lane l of a 16-lane group hands in row l / 4, columns 4 (l % 4) .. + 3 and gets column l of the four rows
    const int half = lane >> 5, sub = lane & 15, colgrp = (lane >> 4) & 1;
    const int rr = r0 + 4 * half + (sub >> 2);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int col = d0 + dt * 32 + colgrp * 16 + 4 * (sub & 3);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf16x8 a;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = rr + 16 * s + 8 * u;
          const char* at = tile + r * TL::ROWB + TL::swizzle(r, col >> 3) * 16 + (col & 7) * 2;
          const bf16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
              (__attribute__((address_space(3))) bf16x4*)(uintptr_t)(uint32_t)(uintptr_t)at);
#pragma unroll
          for (int e = 0; e < 4; ++e) a[4 * u + e] = t[e];
        }
        acc[dt] = Type<__bf16>::mma(a, b[s], acc[dt]);
      }
    }
  }
};
template <int DP, int DT>
struct ColumnProduct<float, DP, DT> {
  static __device__ __forceinline__ void run(const char* tile, int r0, int d0, const float (&p)[16], f32x16 (&acc)[DT], int lane) {
    using TL = Tile<float, DP>;
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = r0 + moving_row(i, half);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int col = d0 + dt * 32 + (lane & 31);
        const float a = *reinterpret_cast<const float*>(tile + r * TL::ROWB + TL::swizzle(r, col >> 2) * 16 + (col & 3) * 4);
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[i], acc[dt], 0, 0, 0);
      }
    }
  }
};

// Rows of a tensor's [.., T, D] slice on their way to an LDS tile: loaded to registers before a tile's arithmetic, written to the
// other buffer after it.  Rows at or past `limit` and masked ones become zero: what lies there (another sequence's values, infinities, NaN)
// must not reach a product, where 0 * NaN would.
template <class T, int DP, int ROWS, int NT = 256>
struct Stage {
  using TL = Tile<T, DP>;
  static constexpr int N = ROWS * TL::NCH / NT, STEP = NT / TL::NCH;
  static_assert(N >= 1 && NT % TL::NCH == 0, "whole rows per pass");
  typename TL::chunk r[N];
  __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, int limit, const uint8_t* mask, int D, bool vec, int tid) {
    const int ch = tid % TL::NCH;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int row = row0 + tid / TL::NCH + n * STEP, rc = min(row, limit - 1);
      typename TL::chunk x = load_chunk<T>(base + rc * stride, ch, D, vec);
      const bool ok = row < limit && !(mask && mask[rc]);
      r[n] = ok ? x : typename TL::chunk{};
    }
  }
  __device__ __forceinline__ void store(char* tile, int tid) const {
    const int ch = tid % TL::NCH;
#pragma unroll
    for (int n = 0; n < N; ++n) TL::put(tile, tid / TL::NCH + n * STEP, ch, r[n]);
  }
};

// A lane's 32 columns x 4 rows of an accumulator as output: column = stationary row, 4 neighbouring d per register group.
template <class T>
__device__ __forceinline__ void store4(T* row, int d, int D, bool vec, float a, float b, float c, float e) {
  const float x[4] = {a, b, c, e};
  if (vec) {  // D is a whole number of chunks, so of fours
    if (d >= D) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4*>(row + d) = f32x4{a, b, c, e};
    } else {
      *reinterpret_cast<bf16x4*>(row + d) = bf16x4{(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)e};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < D) row[d + i] = (T)x[i];
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

// The bias of head h by clamped distance, in log2 units: lut[rel + max_distance].  Finite values below -1e30 become -1e30: the
// same softmax in 32 bits (nothing a score can add is left at either size), without overflow in the change of unit.
__device__ __forceinline__ void fill_lut(const Params& p, int h, float* lut, int tid, int threads) {
  for (int i = tid; i <= 2 * p.max_distance; i += threads) {
    float x = p.table[(int64_t)bucket_of(p, i - p.max_distance) * p.H + h];
    if (x < -1e30f && x >= -3.4028235e38f) x = -1e30f;
    lut[i] = x * kLog2e;
  }
}

// s (raw products of one 32-key subtile) -> scores in log2 units with bias, and -inf where a pair is left out.
// key0: first key of the subtile; pos: the lane's query position; add: 0 / -inf by key, from LDS, or null.
template <bool BIAS>
__device__ __forceinline__ void finish_scores(const Params& p, const f32x16& raw, float (&s)[16], int key0, int pos, int pos_lo, int pos_hi,
                                              const float* add, const float* lut, int half) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    f32x4 km = {};
    if (add) km = *reinterpret_cast<const f32x4*>(add + 8 * g + 4 * half);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[4 * g + e] = raw[4 * g + e] * p.scale2 + km[e];
  }
  if constexpr (BIAS) {
    const int md = p.max_distance;
    if (key0 + 31 - pos_lo <= -md || key0 - pos_hi >= md) {
      const float far = lut[key0 - pos_hi >= md ? 2 * md : 0];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] += far;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] += lut[min(max(key0 + moving_row(i, half) - pos, -md), md) + md];
    }
  }
  if (p.causal && key0 + 31 > pos_lo) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (key0 + moving_row(i, half) > pos) s[i] = -INFINITY;
  }
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

// Work item of a workgroup: consecutive items go to one XCD (workgroups are dealt to the eight XCDs in turn), so that the tiles of
// one head share an L2.  Launch 8 * ceil(n / 8) workgroups; a result >= n has nothing to do.
__device__ __forceinline__ int xcd_item(int n) {
  const int per = (n + 7) >> 3;
  return (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
}

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
static int launch(K kernel, std::atomic<uint64_t>* done, int64_t items, size_t lds, const Params& p, hipStream_t st) {
  if (allow_lds(kernel, done)) return 1;
  WRNN_REQUIRE(lds <= kLdsBytes, "attention: %zu bytes of LDS", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(8 * ((items + 7) / 8))), dim3(256), lds, st, p);
  WRNN_LAUNCH_CHECK();
  return 0;
}

// Whether every row of a [B, H, T, D] tensor starts on 16 bytes.
static inline bool rows_on_16(const void* ptr, int64_t b, int64_t h, int64_t t, int es) {
  return ((reinterpret_cast<uintptr_t>(ptr) | (uintptr_t)(b * es) | (uintptr_t)(h * es) | (uintptr_t)(t * es)) & 15) == 0;
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
