// Self-attention, backward.  With P recomputed from the forward pass's row statistics, P = exp2(score - m) / l:
//   dv = P^T dout,  dP = dout v^T,  delta = rowsum(dout * out),  dS = P * (dP - delta),  dq = scale * dS k,  dk = scale * dS^T q,
//   dtable[n, h] = sum of dS over the pairs whose distance falls in bucket n.
//
// Two kernels, each with its own output rows stationary, so that every sum has one owner and one order (no atomics: the same
// inputs give the same bits): dq walks the keys, dk / dv walk the queries of all heads that share them.  Seven tile products
// in place of the five of a form that adds dq up in memory.
//
// Bound by the matrix instructions (the rates count all seven products):
//   bfloat16  2 x 16 heads, 4096 x 4096 x 128  1291 us  745 TFLOP/s (a library product of 8192 x 8192 x 8192: 1173)
//                                     x 64      629 us  764, and the eighth product of dS's second plane
//             2 x 8 heads,  4096 x 4096 x 256  2459 us  391
//   float32   2 x 16 heads, 2048 x 2048 x 128  1317 us  183 (six partial products: 195 is the library product's sixth)
//                                     x 64      663 us  181
//             2 x 8 heads,  2048 x 2048 x 256  1749 us  138
// Past 128 columns one tile buffer is all that fits in float32, so its conversion is not hidden, and the two waves of a row meet twice a round.
#pragma once
#include "attention_tile.h"

namespace wrnn {
namespace attn {

// The position table's share of a 32 x 32 tile of dS (column: key, the lane's 16 rows: queries), added to the wave's `sums` by distance.  The
// tile goes through LDS 16 keys at a time, skewed: a row of `skew` is a diagonal, its 16 words the keys; words off the tile stay zero, so one
// lane adds one diagonal up in wide reads without a condition.  (Adding each element to `sums` by an LDS add took twice as long as everything else
// of the kernel.)  Distances past max_distance share its bucket: whole tiles of them go to the lane's two registers, the others' to PAD words beside
// the table, which the end folds in.
struct BiasGrad {
  static constexpr int PAD = 64;  // a tile that reaches past max_distance does so by at most 62
  static constexpr int LD = 20, SKEW = 48 * LD;  // 47 diagonals of 16 keys, and one that stays zero
  float below = 0.f, above = 0.f;
  static __host__ __device__ int words(int md) { return (2 * md + 1 + 2 * PAD + 3) & ~3; }
  // rel0: first key - position of the first query
  __device__ __forceinline__ void add(const float (&ds)[16], int rel0, int md, float* skew, float* sums, int lane) {
    const int half = lane >> 5, col = lane & 31;
    if (rel0 + 31 <= -md || rel0 - 31 >= md) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) x += ds[i];
      if (rel0 < 0) below += x;
      else above += x;
      return;
    }
    float* to = skew + (15 - (col & 15) + 4 * half) * LD + (col & 15);
    f32x4 x[8];
#pragma unroll
    for (int n = 0; n < 2; ++n) {  // keys 16 n ..; a wave's LDS instructions keep their order
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (col >> 4 == n)
#pragma unroll
        for (int i = 0; i < 16; ++i) to[moving_row(i, 0) * LD] = ds[i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const int d = n ? lane : lane - 16;  // of distance rel0 + 31 - lane
      const f32x4* row = reinterpret_cast<const f32x4*>(skew + (d >= 0 && d < 47 ? d : 47) * LD);
#pragma unroll
      for (int c = 0; c < 4; ++c) x[4 * n + c] = row[c];
    }
    const f32x4 y = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    if (lane < 63) sums[PAD + md + rel0 + 31 - lane] += (y[0] + y[1]) + (y[2] + y[3]);
  }
  // the wave's sums at distances -md .. md, from sums[PAD] on
  __device__ __forceinline__ void fold(int md, float* sums, int lane) {
    below += sums[lane];
    above += sums[PAD + 2 * md + 1 + lane];
    for (int m = 1; m < 64; m <<= 1) {
      below += __shfl_xor(below, m);
      above += __shfl_xor(above, m);
    }
    if (lane == 0) {
      sums[PAD] += below;
      sums[PAD + 2 * md] += above;
    }
    below = above = 0.f;
  }
};

// A workgroup: 4 waves against every subtile of a tile.  Up to 128 columns each has 32 stationary rows of its own; with more, both sums and both
// stationary operands of a wave would not fit its registers, and two waves share 32 rows, each with half of the columns: of the scores' and dP's
// sums they exchange their parts through LDS.
template <class T, int DP>
struct BackwardShape {
  static constexpr int NP = Type<T>::NP;
  static constexpr int THREADS = 256, NS = NP == 1 && DP < 256 ? 2 : 1, BM = 32 * NS;
  static constexpr int BUFS = NP == 3 && DP == 256 ? 1 : 2;  // two where they leave room for the position bias's tables
  static constexpr bool EARLY = NP == 3 && BUFS == 2;        // the next tile goes to LDS beside the arithmetic (forward pass)
  static constexpr int SLICES = DP > 128 ? 2 : 1, RG = 4 / SLICES, ROWS = 32 * RG;  // waves of a row; groups of 32 rows
  static constexpr int DA = DP / SLICES, DT = DA / 32, NC2 = DA / 16;               // a wave's columns
  static constexpr bool RAW = NP == 3 && SLICES > 1;  // of dk, dv: their two sums leave no room for the planes
  using TL = Tile<T, DP, BM>;
  static constexpr size_t EXCHANGE = SLICES > 1 ? 4 * 16 * 64 * 4 : 0, TILES = 2 * BUFS * TL::BYTES + EXCHANGE;
  static constexpr int WAVES = DP * NP <= 64 ? 2 : 1;  // per SIMD
  // dS of the dq kernel in bfloat16.  A query's keys share the shift along it that its softmax gives them, and the errors of dS add up along it,
  // the more so the fewer columns there are: with one plane dq is off by 2.5e-3 .. 3.3e-3 of its norm up to 64 columns, by 2.4e-3 .. 2.9e-3 above,
  // the most where a query has few keys (rounding dq itself: 1.7e-3).  With two, 1.7e-3 .. 2.1e-3: always up to 64 columns (2 x 16 heads,
  // 4096 x 4096: 541 -> 611 us), above that, where the matrix instructions bound the kernel (1253 -> 1407 us), only for blocks of queries that
  // reach at most FEW keys.
  static constexpr bool FINE = NP == 1 && DP == 64;
  template <int BIAS>
  static constexpr bool CORRECTED = BIAS == 2 || NP == 1;  // of delta (attention_dq_kernel)
  static constexpr int FEW = 1024;
};

// Both waves' parts of a sum added up.  `mine` and `other` are the waves' places; what a wave hands in stays until the other has read it, so the
// next sum goes the other way round, into the place that only this wave reads from.
__device__ __forceinline__ void exchange(f32x16& x, float* mine, const float* other, int lane) {
#pragma unroll
  for (int g = 0; g < 4; ++g) *reinterpret_cast<f32x4*>(mine + (g * 64 + lane) * 4) = f32x4{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
  __syncthreads();
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(other + (g * 64 + lane) * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * g + e] += y[e];
  }
}

// A lane's sums to its row: of the gradient, or (part) of the workgroup's share in 32 bits, which attention_share_kernel adds up.
template <class S, class T>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[S::DT], T* row, float* part, int d0, int D, float scale, int half) {
#pragma unroll
  for (int dt = 0; dt < S::DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = column_of<T>(d0 + dt * 32 + 8 * g + 4 * half, D);
      const float x[4] = {acc[dt][4 * g] * scale, acc[dt][4 * g + 1] * scale, acc[dt][4 * g + 2] * scale, acc[dt][4 * g + 3] * scale};
      if (part) store4<float>(part, d, D, x[0], x[1], x[2], x[3]);
      else store4<T>(row, d, D, x[0], x[1], x[2], x[3]);
    }
}

// The two products of a float32 round (scores, and dP), with the next tiles' conversion in their shadow.
template <class TL, int NC2, class ST, class STAGE>
__device__ __forceinline__ void products_shadow(const char* x, const char* y, const ST& u, const ST& v, f32x16& raw, f32x16& dp, STAGE& sx, STAGE& sy,
                                                char* xn, char* yn, int col, int half, int tid) {
  Splitter sp;
  constexpr int PIECES = STAGE::PIECES;
  const auto piece = [&](int i) {
    if (i < PIECES) sx.store_piece(xn, tid, i, sp);
    else sy.store_piece(yn, tid, i - PIECES, sp);
  };
  Operand<float> a0 = TL::row_chunk(x, col, half), a1 = TL::row_chunk(y, col, half);
#pragma unroll
  for (int c = 0; c < NC2; ++c) {
    Operand<float> n0 = a0, n1 = a1;
    if (c + 1 < NC2) n0 = TL::row_chunk(x, col, 2 * c + 2 + half), n1 = TL::row_chunk(y, col, 2 * c + 2 + half);
    mma2(a0, u.get(c), raw, a1, v.get(c), dp, [&](int m) { shadow<12 * NC2, 2 * PIECES>(12 * c + m, piece); });
    a0 = n0, a1 = n1;
  }
}

// dq: queries stationary, key tiles through LDS.  delta = rowsum(dout * out) carries the rounding of out and of the probabilities behind it.  The table's
// gradient adds it up over all rows in the buckets that hold most of a row's keys, and in bfloat16 dk shows it: with few keys (2.8e-3 of its
// norm, without 2.4e-3), and at any length where the values lie far from zero beside their spread (30 +- 1: 3 .. 6e-2, without 2.4e-3).
// There the kernel also sums dS over each row - what delta is off by, as the probabilities add up to one - and the next kernel, which makes dk, dv and the
// table's gradient, works with the corrected delta, the sum of the shares' planes: a second walk over the keys for it took twice the
// time.  dq itself keeps the uncorrected delta, and is off by 4e-2 .. 1e-1 of its norm with such values.
template <class T, int DP, int BIAS>
__global__ __launch_bounds__(256, (BackwardShape<T, DP>::WAVES)) void attention_dq_kernel(Params p) {
  using S = BackwardShape<T, DP>;
  using TL = typename S::TL;
  constexpr int BN = S::BM, NC2 = S::NC2, BUFS = S::BUFS, NT = S::THREADS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* kt = smem;
  char* vt = smem + BUFS * TL::BYTES;
  int* word = reinterpret_cast<int*>(smem + S::TILES);
  float* lut = reinterpret_cast<float*>(word + 4);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = (p.Tq + S::ROWS - 1) / S::ROWS;
  const Item item(p.B * p.H, nt, p.dq_splits, p.causal);
  if (item.share < 0) return;
  const int share = item.share, d0 = wave % S::SLICES * S::DA, ch0 = d0 / 8;  // the wave's first column, and its chunk
  float* place = reinterpret_cast<float*>(smem + S::TILES - S::EXCHANGE);
  float *mine = place + wave * 1024, *other = place + (wave ^ 1) * 1024;
  const int bh = item.head, b = bh / p.H, h = bh - b * p.H, qt = p.causal ? nt - 1 - item.tile : item.tile;
  const int q0 = qt * S::ROWS + 32 * (wave / S::SLICES);
  const int off = start_of(p, b), kvh = h / p.group;
  const T* kb = reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h;
  const T* vb = reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h;
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  const int qi = q0 + col, qc = min(qi, p.Tq - 1), pos = qi + off;
  const int pos_lo = q0 + off, pos_hi = pos_lo + 31;
  // a query without keys (or past the last one) takes part in nothing, whatever its q and dout hold
  RowStats row;
  row.load(p, (int64_t)bh * p.Tq + qi, qi < p.Tq);
  const float m = row.m(), inv = row.inv();  // 1 / l enters where the sums over the keys are stored
  Stationary<T, S::DA, false> q, go;
  float delta = 0.f;
  {
    const T* gr = reinterpret_cast<const T*>(p.dout) + b * p.do_b + h * p.do_h + qc * p.do_t;
    q.load(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h + qc * p.q_t + d0, half, p.D - d0, row.some(), p.flip);
    go.load(gr + d0, half, p.D - d0, row.some());
    const T* orow = reinterpret_cast<const T*>(p.o_in) + b * p.oi_b + h * p.oi_h + qc * p.oi_t;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const Raw<T> g = load_chunk<T>(gr, 2 * c + half, p.D), o = load_chunk<T>(orow, 2 * c + half, p.D);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)g.x[e] * (float)o.x[e];
    }
    delta = row.some() ? both_sum(delta) : 0.f;
  }
  if constexpr (BIAS != 0) fill_lut(p, h, lut, tid, NT);
  const int end = key_end(p, b, min(qt * S::ROWS + S::ROWS - 1, p.Tq - 1) + off, word, tid, NT);
  const int all = (end + BN - 1) / BN, per = (all + p.dq_splits - 1) / p.dq_splits;
  f32x16 acc[S::DT] = {};
  float off_by = 0.f;
  Stage<T, DP, BN, NT> sk, sv;
  sk.start(kb, p.k_t, end, p.D, tid);
  sv.start(vb, p.v_t, end, p.D, tid);
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
  // the order of a round: as in the forward pass
  const int t0 = share * per, t1 = min(all, t0 + per);
  KeyBits<BN> keys(mask, end, lane, t0 * BN);
  RowBits use = keys.next(t0 * BN), use1 = keys.next((t0 + 1) * BN), use2;  // of tiles t, t + 1, t + 2
  load(t0, use);
  store(t0, use);
  if (S::EARLY) load(t0 + 1, use1);
  __syncthreads();
  auto walk = [&](auto few) {
    constexpr bool exact = decltype(few)::value;
    for (int t = t0; t < t1; ++t) {
      const char *kk = kt + (t & (BUFS - 1)) * TL::BYTES, *vv = vt + (t & (BUFS - 1)) * TL::BYTES;
      use2 = keys.next((t + 2) * BN);
      if (!S::EARLY) load(t + 1, use1);
#pragma unroll
      for (int x = 0; x < S::NS; ++x) {
        const int sub = x, key0 = t * BN + sub * 32;
        const bool work = key0 < end && !(p.causal && key0 > pos_hi);
        f32x16 raw = {}, dp = {};
        if constexpr (S::EARLY) {
          char *kn = kt + ((t + 1) & (BUFS - 1)) * TL::BYTES, *vn = vt + ((t + 1) & (BUFS - 1)) * TL::BYTES;
          products_shadow<TL, NC2>(kk, vv, q, go, raw, dp, sk, sv, kn, vn, col, half, tid);
          load(t + 2, use2);
        } else if (work) {
#pragma unroll
          for (int c = 0; c < NC2; ++c)
            mma2(TL::row_chunk(kk, sub * 32 + col, ch0 + 2 * c + half), q.get(c), raw, TL::row_chunk(vv, sub * 32 + col, ch0 + 2 * c + half), go.get(c),
                 dp, [](int) {});
        }
        if constexpr (S::SLICES > 1) {
          exchange(raw, mine, other, lane);
          exchange(dp, other, mine, lane);
        }
        if (S::EARLY || work) {
          float pr[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pr[i] = raw[i];
          finish_scores<BIAS != 0>(p, pr, key0, pos, pos_lo, pos_hi, use.of(sub), lut, half);
#pragma unroll
          for (int i = 0; i < 16; ++i) pr[i] = __builtin_amdgcn_exp2f(exponent<BIAS != 0>(p, pr[i], m));
#pragma unroll
          for (int i = 0; i < 16; ++i) pr[i] *= dp[i] - delta;
          if constexpr (S::template CORRECTED<BIAS>)
#pragma unroll
            for (int i = 0; i < 16; ++i) off_by += pr[i];
          if constexpr (S::EARLY)
            column_product_shadow<TL, S::DT, 0>(kk, 0, d0, [&](int i) { return pr[i]; }, acc, lane, nullptr, [](int) {});
          else
            column_product<T, TL>(kk, sub * 32, d0, std::conditional_t<S::FINE || exact, Weights2, Weights<T>>(pr), acc, lane);
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
  };
  // (two loops: a choice inside would have both its ways' sums copied in every round)
  if constexpr (S::NP == 1 && !S::FINE) {
    if (end <= S::FEW) walk(std::true_type());
    else walk(std::false_type());
  } else {
    walk(std::false_type());
  }
  off_by = both_sum(off_by) * inv;
  if (half == 0 && d0 == 0 && qi < p.Tq && (S::template CORRECTED<BIAS> || share == 0))
    p.delta[((int64_t)share * p.B * p.H + bh) * p.Tq + qi] = share == 0 ? delta + off_by : off_by;
  if (qi < p.Tq)
    store_rows<S>(acc, reinterpret_cast<T*>(p.dq) + b * p.dq_b + h * p.dq_h + qi * p.dq_t,
                  p.dq_splits > 1 ? p.dq_part + (((int64_t)share * p.B * p.H + bh) * p.Tq + qi) * p.D : nullptr, d0, p.D, p.scale * inv, half);
}

// dk, dv and, with BIAS == 2, the position table's gradient: keys of one key head stationary; tiles of queries and their output gradients through
// LDS, over all heads of the group.
template <class T, int DP, int BIAS>
__global__ __launch_bounds__(256, (BackwardShape<T, DP>::WAVES)) void attention_dkv_kernel(Params p) {
  using S = BackwardShape<T, DP>;
  using TL = typename S::TL;
  constexpr int BM = S::BM, NC2 = S::NC2, BUFS = S::BUFS, NT = S::THREADS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* qt = smem;
  char* gt = smem + BUFS * TL::BYTES;
  float* stat = reinterpret_cast<float*>(smem + S::TILES);  // [BUFS][3][BM]: m, 1 / l, delta
  float* lut = stat + BUFS * 3 * BM;
  const int words = BiasGrad::words(p.max_distance);
  float* skew = lut + ((2 * p.max_distance + 4) & ~3);
  float* sums = skew + S::RG * BiasGrad::SKEW;  // [RG][words]
  BiasGrad bias_grad;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = (p.Tk + S::ROWS - 1) / S::ROWS;
  const Item item(p.B * p.Hkv, nt, p.dkv_splits, p.causal);
  if (item.share < 0) return;
  const int share = item.share, d0 = wave % S::SLICES * S::DA, ch0 = d0 / 8, rg = wave / S::SLICES;
  float* place = reinterpret_cast<float*>(smem + S::TILES - S::EXCHANGE);
  float *mine = place + wave * 1024, *other = place + (wave ^ 1) * 1024;
  const int bh = item.head, b = bh / p.Hkv, kvh = bh - b * p.Hkv, k0 = item.tile * S::ROWS, kw = k0 + 32 * rg;
  const int off = start_of(p, b), key = kw + col, kc = min(key, p.Tk - 1);
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  int end = p.Tk;
  if (p.key_lens) end = min(end, max(p.key_lens[b], 0));
  if (p.causal) end = min(end, max(p.Tq + off, 0));  // past the last query's reach
  const bool ok = key < end && !(mask && mask[kc]);
  Stationary<T, S::DA, S::RAW> k, v;
  k.load(reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h + kc * p.k_t + d0, half, p.D - d0, ok, p.flip);
  v.load(reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h + kc * p.v_t + d0, half, p.D - d0, ok);
  f32x16 dk[S::DT] = {}, dv[S::DT] = {};
  // under causality queries before key - off see nothing of this block
  const int qt_n = (p.Tq + BM - 1) / BM, qt_0 = p.causal ? min(max(k0 - off, 0) / BM, qt_n) : 0, per = qt_n - qt_0;
  const int all = k0 < end ? per * p.group : 0, part = (all + p.dkv_splits - 1) / p.dkv_splits, first_it = share * part,
            steps = min(all, first_it + part);
  Stage<T, DP, BM, NT> sq, sg;
  sq.start(nullptr, p.q_t, p.Tq, p.D, tid);
  sg.start(nullptr, p.do_t, p.Tq, p.D, tid);
  RowStats s_row = {};  // lane's row of the tile on its way
  float s_delta = 0.f;
  bool there = false;
  auto load = [&](int it) {
    if (it >= steps) return;
    const int h = kvh * p.group + it / per, r0 = (qt_0 + it % per) * BM;
    there = lane < BM && r0 + lane < p.Tq;
    const int64_t row = ((int64_t)b * p.H + h) * p.Tq + r0 + lane;
    s_row.load(p, row, there);
    sq.base = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h);
    sg.base = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.dout) + b * p.do_b + h * p.do_h);
    sq.load(r0, nullptr, tid);
    sg.load(r0, nullptr, tid);
    if (tid < BM) {
      s_delta = 0.f;
      if (there)
        for (int n = 0; n < (S::template CORRECTED<BIAS> ? p.dq_splits : 1); ++n) s_delta += p.delta[(int64_t)n * p.B * p.H * p.Tq + row];
    }
  };
  auto store_stat = [&](int it) {
    const int o = it & (BUFS - 1);
    if (tid < BM) {
      stat[o * 3 * BM + tid] = s_row.m();
      stat[(o * 3 + 1) * BM + tid] = s_row.inv();
      stat[(o * 3 + 2) * BM + tid] = s_row.some() ? s_delta : 0.f;
    }
  };
  // Queries without keys: their rows become zero on their way to LDS.  P = 0 alone would not keep out what they hold, 0 * NaN being NaN.
  auto drop = [&]() {
    const uint64_t none = __ballot(there && !s_row.some());
    if (none) {
      RowBits use;
      use.lo = ~none;
      sq.drop(use, tid);
      sg.drop(use, tid);
    }
  };
  auto store = [&](int it) {
    const int o = it & (BUFS - 1);
    drop();
    sq.store(qt + o * TL::BYTES, tid);
    sg.store(gt + o * TL::BYTES, tid);
    store_stat(it);
  };
  if (BIAS == 2)
    for (int i = tid; i < S::RG * BiasGrad::SKEW; i += NT) skew[i] = 0.f;
  load(first_it);
  store(first_it);
  if (S::EARLY) load(first_it + 1);
  __syncthreads();
  for (int it = first_it; it < steps; ++it) {
    if constexpr (BIAS) {
      if (it == first_it || it % per == 0) {
        fill_lut(p, kvh * p.group + it / per, lut, tid, NT);
        if (BIAS == 2)
          for (int i = tid; i < S::RG * words; i += NT) sums[i] = 0.f;
        __syncthreads();
      }
    }
    const int o = it & (BUFS - 1), r0 = (qt_0 + it % per) * BM;
    const char *qq = qt + o * TL::BYTES, *gg = gt + o * TL::BYTES;
    if (!S::EARLY) load(it + 1);
#pragma unroll
    for (int x = 0; x < S::NS; ++x) {
      const int sub = x, i0 = r0 + sub * 32, p0 = i0 + off;  // position of the subtile's first query
      const bool work = kw < end && i0 < p.Tq && !(p.causal && kw > p0 + 31);
      f32x16 raw = {}, dp = {};
      if constexpr (S::EARLY) {
        char *qn = qt + ((it + 1) & (BUFS - 1)) * TL::BYTES, *gn = gt + ((it + 1) & (BUFS - 1)) * TL::BYTES;
        drop();
        products_shadow<TL, NC2>(qq, gg, k, v, raw, dp, sq, sg, qn, gn, col, half, tid);
        store_stat(it + 1);
        load(it + 2);
      } else if (work) {
#pragma unroll
        for (int c = 0; c < NC2; ++c)
          mma2(TL::row_chunk(qq, sub * 32 + col, ch0 + 2 * c + half), k.get(c), raw, TL::row_chunk(gg, sub * 32 + col, ch0 + 2 * c + half), v.get(c), dp,
               [](int) {});
      }
      if constexpr (S::SLICES > 1) {
        exchange(raw, mine, other, lane);
        exchange(dp, other, mine, lane);
      }
      if (S::EARLY || work) {
        float s[16];
        if constexpr (BIAS) {
          const int md = p.max_distance;
          if (kw + 31 - p0 <= -md || kw - (p0 + 31) >= md) {
            const float far = ok ? lut[kw > p0 ? 2 * md : 0] : -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = fmaf(raw[i], p.scale2, far);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = fmaf(raw[i], p.scale2, ok ? lut[min(max(key - p0 - moving_row(i, half), -md), md) + md] : -INFINITY);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = raw[i];
        }
        const float* of = stat + o * 3 * BM + sub * 32 + 4 * half;
        float ds[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 m = *reinterpret_cast<const f32x4*>(of + 8 * g), inv = *reinterpret_cast<const f32x4*>(of + BM + 8 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * g + e] = __builtin_amdgcn_exp2f(exponent<BIAS != 0>(p, s[4 * g + e], m[e])) * inv[e];
        }
        if (p.causal && kw + 31 > p0) {
          const int first = key - p0 - 4 * half;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = first > moving_row(i, 0) ? 0.f : s[i];
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 de = *reinterpret_cast<const f32x4*>(of + 2 * BM + 8 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) ds[4 * g + e] = s[4 * g + e] * (dp[4 * g + e] - de[e]);
        }
        if constexpr (BIAS == 2)
          if (d0 == 0) bias_grad.add(ds, kw - p0, p.max_distance, skew + rg * BiasGrad::SKEW, sums + rg * words, lane);
        if constexpr (S::EARLY) {
          Splitter first;  // of dS, made beside the products with P
          column_product_shadow<TL, S::DT, 12>(gg, 0, d0, [&](int i) { return s[i]; }, dv, lane, nullptr,
                                               [&](int i) { first.step(i, [&](int n) { return ds[n]; }); });
          column_product_shadow<TL, S::DT, 0>(qq, 0, d0, [&](int i) { return ds[i]; }, dk, lane, &first, [](int) {});
        } else {
          column_product<T, TL>(gg, sub * 32, d0, Weights<T>(s), dv, lane);
          column_product<T, TL>(qq, sub * 32, d0, Weights<T>(ds), dk, lane);
        }
      }
    }
    if (!S::EARLY) {
      if (BUFS == 1) __syncthreads();
      store(it + 1);
    }
    __syncthreads();
    if constexpr (BIAS == 2) {
      if (it + 1 == steps || (it + 1) % per == 0) {  // the end of a head: the waves' sums, then a bucket's distances, in a fixed order
        if (d0 == 0) bias_grad.fold(p.max_distance, sums + rg * words, lane);
        __syncthreads();
        for (int i = tid; i < words; i += NT) {
          float x = sums[i];
          for (int w = 1; w < S::RG; ++w) x += sums[w * words + i];
          sums[i] = x;
        }
        __syncthreads();
        const int64_t row = (int64_t)(b * nt + item.tile) * p.dkv_splits + share;
        for (int i = tid; i < p.buckets; i += NT) p.dtable_part[(row * p.H + kvh * p.group + it / per) * p.buckets + i] = bucket_sum(p, sums + BiasGrad::PAD, i);
        __syncthreads();
      }
    }
  }
  if constexpr (BIAS == 2) {
    for (int g = 0; g < p.group; ++g)  // heads that this share has nothing of
      if (first_it >= steps || g < first_it / per || g > (steps - 1) / per) {
        const int64_t row = (int64_t)(b * nt + item.tile) * p.dkv_splits + share;
        for (int i = tid; i < p.buckets; i += NT) p.dtable_part[(row * p.H + kvh * p.group + g) * p.buckets + i] = 0.f;
      }
    if (!p.dk) return;
  }
  T* kout = reinterpret_cast<T*>(p.dk) + b * p.dk_b + kvh * p.dk_h;
  T* vout = reinterpret_cast<T*>(p.dv) + b * p.dv_b + kvh * p.dv_h;
  if (!ok) {  // left out: what the loop added up there is no probability
#pragma unroll
    for (int dt = 0; dt < S::DT; ++dt) dk[dt] = f32x16{}, dv[dt] = f32x16{};
  }
  if (key < p.Tk) {
    float* to = nullptr;
    const int64_t rows = (int64_t)p.B * p.Hkv * p.Tk;
    if (p.dkv_splits > 1) to = p.dkv_part + (share * 2 * rows + (int64_t)bh * p.Tk + key) * p.D;
    store_rows<S>(dk, kout + key * p.dk_t, to, d0, p.D, p.scale, half);
    store_rows<S>(dv, vout + key * p.dv_t, to ? to + rows * p.D : nullptr, d0, p.D, 1.f, half);
  }
}

// The workgroups' shares added up in their order: out[b, h, t, :] = sum over s of part[s][(b H + h) T + t][:].  blockIdx.y: dk, dv.
template <class T>
__global__ __launch_bounds__(256) void attention_share_kernel(const float* part, int splits, int64_t step, int64_t pair, int64_t rows, int T_, int H, int D, T* out0,
                                                              T* out1, int64_t b0, int64_t h0, int64_t t0, int64_t b1, int64_t h1, int64_t t1) {
  const int quads = D / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / quads;
  if (row >= rows) return;
  const int d = (int)(i - row * quads) * 4;
  const float* x = part + blockIdx.y * pair + row * D + d;
  f32x4 s = *reinterpret_cast<const f32x4*>(x);
  for (int n = 1; n < splits; ++n) s += *reinterpret_cast<const f32x4*>(x + n * step);
  const int t = row % T_;
  const int64_t bh = row / T_, b = bh / H, h = bh % H;
  T* o = blockIdx.y ? out1 + b * b1 + h * h1 + t * t1 : out0 + b * b0 + h * h0 + t * t0;
  store4<T>(o, d, D, s[0], s[1], s[2], s[3]);
}

// ------------------------------------------------------------------ host

template <class T, int DP, int BIAS>
static int launch_backward(const Params& p, float* dtable, hipStream_t st) {
  using S = BackwardShape<T, DP>;
  static std::atomic<uint64_t> dq_done{0}, dkv_done{0};
  const size_t lut = BIAS ? (size_t)(2 * p.max_distance + 4) * 4 : 0;
  const int k_tiles = (p.Tk + S::ROWS - 1) / S::ROWS;
  if (launch(&attention_dq_kernel<T, DP, BIAS>, &dq_done, (int64_t)p.B * p.H * ((p.Tq + S::ROWS - 1) / S::ROWS) * p.dq_splits, S::THREADS,
             S::TILES + 16 + lut, p, st))
    return 1;
  if (p.dq_splits > 1) {
    const int64_t rows = (int64_t)p.B * p.H * p.Tq;
    T* dq = static_cast<T*>(p.dq);
    hipLaunchKernelGGL((attention_share_kernel<T>), dim3((unsigned)((rows * (p.D / 4) + 255) / 256)), dim3(256), 0, st, p.dq_part, p.dq_splits, rows * p.D,
                       int64_t(0), rows, p.Tq, p.H, p.D, dq, dq, p.dq_b, p.dq_h, p.dq_t, p.dq_b, p.dq_h, p.dq_t);
    WRNN_LAUNCH_CHECK();
  }
  if ((p.dk || BIAS == 2) && p.Tk) {
    if (launch(&attention_dkv_kernel<T, DP, BIAS>, &dkv_done, (int64_t)p.B * p.Hkv * k_tiles * p.dkv_splits, S::THREADS,
               S::TILES + S::BUFS * 3 * S::BM * 4 + lut + (BIAS == 2 ? (size_t)S::RG * (BiasGrad::SKEW + BiasGrad::words(p.max_distance)) * 4 : 0), p, st))
      return 1;
    if (p.dk && p.dkv_splits > 1) {
      const int64_t rows = (int64_t)p.B * p.Hkv * p.Tk;
      hipLaunchKernelGGL((attention_share_kernel<T>), dim3((unsigned)((rows * (p.D / 4) + 255) / 256), 2), dim3(256), 0, st, p.dkv_part, p.dkv_splits,
                         2 * rows * p.D, rows * p.D, rows, p.Tk, p.Hkv, p.D, static_cast<T*>(p.dk), static_cast<T*>(p.dv), p.dk_b, p.dk_h, p.dk_t, p.dv_b,
                         p.dv_h, p.dv_t);
      WRNN_LAUNCH_CHECK();
    }
  }
  if (BIAS == 2) return launch_table_sum<float>(p.dtable_part, p.B * k_tiles * p.dkv_splits, p.H, p.buckets, dtable, st);
  return 0;
}

template <class T, int DP>
int backward(const Params& p, float* dtable, hipStream_t st) {
  return !p.table ? launch_backward<T, DP, 0>(p, dtable, st) : dtable ? launch_backward<T, DP, 2>(p, dtable, st) : launch_backward<T, DP, 1>(p, dtable, st);
}

}  // namespace attn
}  // namespace wrnn
