// Self-attention, forward:  out = softmax(scale * q k^T + bias) v  over the keys that lengths, mask and causality leave.
//
// One pass over the keys with a running maximum and sum per query (kept in 32 bits, in units of log2 so that the exponential is
// one v_exp_f32).  The [Tq, Tk] scores only ever exist as 32 x 32 tiles in registers (attention_tile.h).
//
// Long sequences are bound by the matrix instructions and, the fewer columns the more, by the softmax's vector instructions between them (bfloat16
// at 128 columns: 120 of those to 16 products a subtile).  Measured, forward only:
//   bfloat16  2 x 16 heads, 4096 x 4096 x 128   291 us  944 TFLOP/s (a library product of 8192 x 8192 x 8192: 1173)
//                                     x 64      173 us  795
//             2 x 8 heads,  4096 x 4096 x 256   412 us  667
//   float32   2 x 16 heads, 2048 x 2048 x 128   354 us  194 (six partial products: 195 is the library product's sixth)
//                                     x 64      178 us  193
//             2 x 8 heads,  2048 x 2048 x 256   445 us  154
// Single tokens over a cache are bound by the reading of it: 8 rows, 16 heads on 4, 8191 keys of 128 columns in bfloat16 31 us, the joining kernel's 4
// included (134 MB at 4.3 TB/s; a large copy moves 4.8); in float32 104 us.
#pragma once
#include "attention_tile.h"

namespace wrnn {
namespace attn {

// Running softmax of one query per lane: maximum, sum (this half-wave's share), and the accumulators it scales.
// The maximum only moves when a score exceeds it by more than 8 (a factor 256, far inside float's range): most tiles rescale nothing.
template <bool BIAS>
struct Running {
  float m = kLowest, l = 0.f;
  template <int NS, int DT>
  __device__ __forceinline__ void move(const Params& p, const float (&s)[NS][16], f32x16 (&acc)[DT]) {
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
    mx = both_max(mx);
    if (!BIAS) mx *= p.scale2;
    if (__builtin_expect(__any(mx > m + 8.f), 0)) {
      const float mn = fmaxf(m, mx), a = exp2f(m - mn);
      m = mn;
      l *= a;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= a;
    }
  }
  __device__ __forceinline__ float weight(const Params& p, float s) {
    const float x = __builtin_amdgcn_exp2f(exponent<BIAS>(p, s, m));
    l += x;
    return x;
  }
};

// Shapes of a workgroup.
//   wide   4 waves, 32 queries each, all against every 32 keys of a tile: a tile in LDS serves 128 queries.
//   narrow 32 query columns, the waves on different 32 keys of a tile, joined at the end; the columns may hold the queries of all heads that
//          share k and v (p.pack).  For single tokens and few queries.  (For more than 32 queries the wide one is the faster also where only a few
//          workgroups run: 32 x 2 heads, 150 x 150 x 64 in float32 17 against 28 us.)
// In either the keys may be divided over workgroups (p.splits), whose sums attention_join_kernel adds up.
template <class T, int DP, bool WIDE>
struct ForwardShape {
  static constexpr int NP = Type<T>::NP;
  // narrow: as many waves as tiles of 32 keys fit the LDS beside each other (three planes of float32 are 6 bytes an element)
  static constexpr int WQ = WIDE ? 4 : 1, WK = WIDE ? 1 : NP == 1 ? 4 : DP == 64 ? 4 : DP == 128 ? 2 : 1;
  static constexpr int NS = WIDE && NP == 1 ? 2 : 1;  // 32-key subtiles of a tile per wave
  // one tile of 32 keys is all that fits: four waves fetch and convert it, of which the last three do the first one's arithmetic for nothing
  static constexpr int COPIES = WQ * WK == 1 ? 4 : 1;
  static constexpr int THREADS = 64 * WQ * WK * COPIES, BN = 32 * WK * NS;
  static constexpr int BUFS = WIDE && !(NP == 3 && DP == 256) ? 2 : 1;  // two where they fit
  static constexpr int WAVES = WIDE ? (DP * NP <= 192 ? 2 : 1) : (DP * NP <= 128 ? 2 : 1);  // per SIMD
  static constexpr bool EARLY = NP == 3 && BUFS == 2;
  static constexpr bool RAW = NP == 3 && DP == 256;
  using TL = Tile<T, DP, BN>;
  static constexpr size_t TILES = 2 * BUFS * TL::BYTES, SUMS = WK > 1 ? (size_t)WK * 32 * (DP + 4) * 4 : 0;
  static constexpr size_t BODY = TILES > SUMS ? TILES : SUMS;
  static constexpr size_t LDS = BODY + 2 * 32 * 4 * 4 + 16;  // + statistics of the waves, a word; the position bias's table follows
};

template <class T, int DP, bool BIAS, bool WIDE>
__global__ __launch_bounds__((ForwardShape<T, DP, WIDE>::THREADS), (ForwardShape<T, DP, WIDE>::WAVES)) void attention_forward_kernel(Params p) {
  using S = ForwardShape<T, DP, WIDE>;
  using TL = typename S::TL;
  constexpr int BN = S::BN, NS = S::NS, NC2 = DP / 16, DT = DP / 32, BUFS = S::BUFS, NT = S::THREADS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* kt = smem;
  char* vt = smem + BUFS * TL::BYTES;
  float* ml = reinterpret_cast<float*>(smem + S::BODY);  // [WK][2][32]
  int* word = reinterpret_cast<int*>(ml + 4 * 2 * 32);
  float* lut = reinterpret_cast<float*>(word + 4);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = WIDE ? wave : 0, wk = WIDE || S::WK == 1 ? 0 : wave;
  const bool pack = !WIDE && p.pack;
  const int heads = pack ? p.Hkv : p.H, splits = p.splits;
  const int nt = pack ? 1 : (p.Tq + 32 * S::WQ - 1) / (32 * S::WQ);
  const Item item(p.B * heads, nt, splits, p.causal);
  if (item.share < 0) return;
  const int part = item.share, bh = item.head, b = bh / heads, hh = bh - b * heads;
  const int q0 = (p.causal ? nt - 1 - item.tile : item.tile) * 32 * S::WQ + 32 * wq;  // under causality the last queries have the longest rows
  const int lh = pack ? col / p.Tq : 0;                                              // the column's head within the group
  const int h = pack ? hh * p.group + min(lh, p.group - 1) : hh, kvh = pack ? hh : hh / p.group;
  const int qi = pack ? col - lh * p.Tq : q0 + col;
  const int off = start_of(p, b), pos = qi + off;
  const int pos_lo = q0 + off, pos_hi = (pack ? p.Tq - 1 : q0 + 31) + off;
  const T* kb = reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h;
  const T* vb = reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h;
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  Stationary<T, DP, S::RAW> q;
  q.load(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h + min(qi, p.Tq - 1) * p.q_t, half, p.D, true, p.flip);
  const int lut_len = 2 * p.max_distance + 1;
  const float* my_lut = lut;
  if constexpr (BIAS) {
    if (pack) {
      for (int g = 0; g < p.group; ++g) fill_lut(p, hh * p.group + g, lut + g * lut_len, tid, NT);
      my_lut += min(lh, p.group - 1) * lut_len;
    } else {
      fill_lut(p, h, lut, tid, NT);
    }
  }
  const int last_pos = min(q0 - 32 * wq + 32 * S::WQ - 1, p.Tq - 1) + off;
  const int end = key_end(p, b, last_pos, word, tid, NT);
  const int all = (end + BN - 1) / BN, per = (all + splits - 1) / splits, t0 = part * per, t1 = min(all, t0 + per);
  f32x16 acc[DT] = {};
  Running<BIAS> run;
  Stage<T, DP, BN, NT> sk, sv;
  sk.start(kb, p.k_t, end, p.D, tid);
  sv.start(vb, p.v_t, end, p.D, tid);
  KeyBits<BN> keys(mask, end, lane, t0 * BN);
  // rows that the mask leaves out: not requested (EARLY), or zeroed on their way to LDS, which keeps the requests one block of code
  auto load = [&](int t, const RowBits& use) {
    sk.load(t * BN, S::EARLY && mask ? &use : nullptr, tid);
    sv.load(t * BN, S::EARLY && mask ? &use : nullptr, tid);
  };
  auto store = [&](int t, const RowBits& use) {
    const int o = t & (BUFS - 1);
    if (!S::EARLY && mask && !use.template all<BN>()) {
      sk.drop(use, tid);
      sv.drop(use, tid);
    }
    sk.store(kt + o * TL::BYTES, tid);
    sv.store(vt + o * TL::BYTES, tid);
  };
  // float32 (EARLY): tile t is worked on while tile t + 1 goes from registers to LDS (its conversion fills the matrix instructions' shadow)
  // and tile t + 2 is requested.  Otherwise tile t + 1 is requested before tile t's arithmetic and goes to LDS after it; with one buffer
  // that waits for everybody to be done with tile t.
  RowBits use = keys.next(t0 * BN), use1 = keys.next((t0 + 1) * BN), use2;  // of tiles t, t + 1, t + 2
  load(t0, use);
  store(t0, use);
  if (S::EARLY) load(t0 + 1, use1);
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const char *kk = kt + (t & (BUFS - 1)) * TL::BYTES, *vv = vt + (t & (BUFS - 1)) * TL::BYTES;
    const int sub0 = NS * wk, key0 = t * BN + 32 * sub0;
    use2 = keys.next((t + 2) * BN);
    if (!S::EARLY) load(t + 1, use1);
    // (EARLY goes without the way round a tile past the wave's reach: joining its two ways costs a copy of every sum in every round)
    if (S::EARLY || (key0 < end && !(p.causal && key0 > pos_hi))) {
      f32x16 raw[NS] = {};
      if constexpr (S::EARLY) {
        char *kn = kt + ((t + 1) & (BUFS - 1)) * TL::BYTES, *vn = vt + ((t + 1) & (BUFS - 1)) * TL::BYTES;
        Splitter sp;
        constexpr int PIECES = decltype(sk)::PIECES;
        const auto piece = [&](int i) {
          if (i < PIECES) sk.store_piece(kn, tid, i, sp);
          else sv.store_piece(vn, tid, i - PIECES, sp);
        };
        auto chunk = [&](int c) { return TL::row_chunk(kk, col, 2 * c + half); };
        f32x16 odd = {};
        Operand<T> a0 = chunk(0), a1 = chunk(1);
#pragma unroll
        for (int c = 0; c < NC2; c += 2) {
          Operand<T> n0 = a0, n1 = a1;
          if (c + 2 < NC2) n0 = chunk(c + 2), n1 = chunk(c + 3);
          mma2(a0, q.get(c), raw[0], a1, q.get(c + 1), odd, [&](int m) { shadow<6 * NC2, 2 * PIECES>(6 * c + m, piece); });
          a0 = n0, a1 = n1;
        }
        raw[0] += odd;
        load(t + 2, use2);
      } else {
#pragma unroll
        for (int c = 0; c < NC2; ++c)
#pragma unroll
          for (int s = 0; s < NS; ++s) raw[s] = mma(TL::row_chunk(kk, (sub0 + s) * 32 + col, 2 * c + half), q.get(c), raw[s]);
      }
      float s[NS][16];
#pragma unroll
      for (int x = 0; x < NS; ++x) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[x][i] = raw[x][i];
        finish_scores<BIAS>(p, s[x], key0 + 32 * x, pos, pos_lo, pos_hi, use.of(sub0 + x), my_lut, half);
      }
      run.move(p, s, acc);
      if constexpr (S::EARLY) {
        column_product_shadow<TL, DT, 0>(vv, 0, 0, [&](int i) { return run.weight(p, s[0][i]); }, acc, lane, nullptr, [](int) {});
      } else {
#pragma unroll
        for (int x = 0; x < NS; ++x) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[x][i] = run.weight(p, s[x][i]);
          column_product<T, TL>(vv, (sub0 + x) * 32, 0, Weights<T>(s[x]), acc, lane);
        }
      }
    }
    if (!S::EARLY) {
      if (BUFS == 1) __syncthreads();
      store(t + 1, use1);
    }
    use = use1;
    use1 = use2;
    __syncthreads();
  }
  const float l = both_sum(run.l);
  if constexpr (S::WK == 1) {
    if (qi >= p.Tq || (pack && lh >= p.group) || (S::COPIES > 1 && wave)) return;
    const int64_t row = ((int64_t)b * p.H + h) * p.Tq + qi;
    if (splits == 1) {
      if (half == 0) store_stats(p, row, run.m, l);
      if (!p.out) return;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      T* orow = reinterpret_cast<T*>(p.out) + b * p.o_b + h * p.o_h + qi * p.o_t;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          store4<T>(orow, column_of<T>(dt * 32 + 8 * g + 4 * half, p.D), p.D, acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv,
                    acc[dt][4 * g + 3] * inv);
    } else {
      float* to = p.part + (row * splits + part) * (DP + 4);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(to + 4 + dt * 32 + 8 * g + 4 * half) = f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
      if (half == 0) {
        to[0] = run.m;
        to[1] = l;
      }
    }
  } else {
    // join the waves: a common maximum per column, then sums over the waves in their order
    if (half == 0) {
      ml[(wk * 2) * 32 + col] = run.m;
      ml[(wk * 2 + 1) * 32 + col] = l;
    }
    __syncthreads();
    float m = ml[col];
#pragma unroll
    for (int w = 1; w < S::WK; ++w) m = fmaxf(m, ml[(w * 2) * 32 + col]);
    const float a = exp2f(run.m - m);
    constexpr int LD = DP + 4;
    float* sums = reinterpret_cast<float*>(smem);  // [WK][32][LD], in the tiles' place
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(sums + (wk * 32 + col) * LD + dt * 32 + 8 * g + 4 * half) =
            f32x4{acc[dt][4 * g] * a, acc[dt][4 * g + 1] * a, acc[dt][4 * g + 2] * a, acc[dt][4 * g + 3] * a};
    __syncthreads();
    constexpr int TPC = NT / 32;  // threads a column
    const int c2 = tid / TPC, d_first = (tid % TPC) * 4;
    float m2 = ml[c2], l2 = 0.f;
#pragma unroll
    for (int w = 1; w < S::WK; ++w) m2 = fmaxf(m2, ml[(w * 2) * 32 + c2]);
#pragma unroll
    for (int w = 0; w < S::WK; ++w) l2 += ml[(w * 2 + 1) * 32 + c2] * exp2f(ml[(w * 2) * 32 + c2] - m2);
    const int lh2 = pack ? c2 / p.Tq : 0, h2 = pack ? hh * p.group + lh2 : hh, qi2 = pack ? c2 - lh2 * p.Tq : q0 + c2;
    if (pack ? lh2 >= p.group : qi2 >= p.Tq) return;
    const int64_t row = ((int64_t)b * p.H + h2) * p.Tq + qi2;
    const float inv = splits > 1 ? 1.f : l2 > 0.f ? 1.f / l2 : (l2 == 0.f ? 0.f : l2);
    T* orow = reinterpret_cast<T*>(p.out) + b * p.o_b + h2 * p.o_h + qi2 * p.o_t;
    float* to = p.part + (row * splits + part) * (DP + 4);
#pragma unroll
    for (int d = d_first; d < DP; d += TPC * 4) {
      f32x4 x = *reinterpret_cast<const f32x4*>(sums + c2 * LD + d);
#pragma unroll
      for (int w = 1; w < S::WK; ++w) x += *reinterpret_cast<const f32x4*>(sums + (w * 32 + c2) * LD + d);
      if (splits > 1)
        *reinterpret_cast<f32x4*>(to + 4 + d) = x;
      else if (p.out)
        store4<T>(orow, column_of<T>(d, p.D), p.D, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    }
    if (d_first == 0) {
      if (splits > 1) {
        to[0] = m2;
        to[1] = l2;
      } else {
        store_stats(p, row, m2, l2);
      }
    }
  }
}

// Joins the splits of a query: one wave per query.  Lane s weighs split s, then the lanes take the columns, splits in their order.
template <class T, int DP>
__global__ __launch_bounds__(256) void attention_join_kernel(Params p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)p.B * p.H * p.Tq) return;
  const float* part = p.part + row * p.splits * (DP + 4);
  float ms = kLowest, ls = 0.f;
  if (lane < p.splits) {
    ms = part[lane * (DP + 4)];
    ls = part[lane * (DP + 4) + 1];
  }
  float m = ms;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) m = fmaxf(m, __shfl_xor(m, i));
  const float w = exp2f(ms - m);
  float l = ls * w;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) l += __shfl_xor(l, i);
  constexpr int E = DP / 64;
  typedef float vec __attribute__((ext_vector_type(E)));
  vec x = vec(0.f);
  for (int s0 = 0; s0 < p.splits; s0 += 8) {  // eight loads in flight; past the last split its own again, weighed zero
    vec y[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) y[u] = *reinterpret_cast<const vec*>(part + min(s0 + u, p.splits - 1) * (DP + 4) + 4 + lane * E);
#pragma unroll
    for (int u = 0; u < 8; ++u) x += y[u] * (s0 + u < p.splits ? __shfl(w, s0 + u) : 0.f);
  }
  if (lane == 0) store_stats(p, row, m, l);
  if (!p.out) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int qi = row % p.Tq, h = (row / p.Tq) % p.H, b = row / p.Tq / p.H;
  T* orow = reinterpret_cast<T*>(p.out) + b * p.o_b + h * p.o_h + qi * p.o_t;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = lane * E + e, d = column_of<T>(c & ~3, p.D);
    if (d >= 0) orow[d + (c & 3)] = (T)(x[e] * inv);
  }
}

template <class T, int DP, bool BIAS>
static int launch_forward(const Params& p, hipStream_t st) {
  static std::atomic<uint64_t> wide_done{0}, narrow_done{0};
  const size_t lut = BIAS ? (2 * p.max_distance + 1) * sizeof(float) : 0;
  if (!p.narrow) {
    using S = ForwardShape<T, DP, true>;
    const int64_t n = (int64_t)p.B * p.H * ((p.Tq + 127) / 128) * p.splits;
    if (launch(&attention_forward_kernel<T, DP, BIAS, true>, &wide_done, n, S::THREADS, S::LDS + lut, p, st)) return 1;
  } else {
    using S = ForwardShape<T, DP, false>;
    const int64_t n = (p.pack ? (int64_t)p.B * p.Hkv : (int64_t)p.B * p.H * ((p.Tq + 31) / 32)) * p.splits;
    if (launch(&attention_forward_kernel<T, DP, BIAS, false>, &narrow_done, n, S::THREADS, S::LDS + lut * (p.pack ? p.group : 1), p, st)) return 1;
  }
  if (p.splits > 1) {
    const int64_t rows = (int64_t)p.B * p.H * p.Tq;
    hipLaunchKernelGGL((attention_join_kernel<T, DP>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
    WRNN_LAUNCH_CHECK();
  }
  return 0;
}

template <class T, int DP>
int forward(const Params& p, hipStream_t st) {
  return p.table ? launch_forward<T, DP, true>(p, st) : launch_forward<T, DP, false>(p, st);
}

}  // namespace attn
}  // namespace wrnn
