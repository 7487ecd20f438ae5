// Self-attention, backward.  With P recomputed from the forward pass's log-sum-exp:
//   dv = P^T dout,  dP = dout v^T,  delta = rowsum(dout * out),  dS = P * (dP - delta),  dq = scale * dS k,  dk = scale * dS^T q,
//   dtable[n, h] = sum of dS over the pairs whose distance falls in bucket n.
//
// Two kernels, each with its own output rows stationary, so that every sum has one owner and one order (no atomics: the same
// inputs give the same bits): dq walks the keys, dk / dv walk the queries of all heads that share them.  Seven tile products
// in place of the five of a form that adds dq up in memory.
#pragma once
#include "attention_tile.h"

namespace wrnn {
namespace attn {

// rel = key - position for the 63 diagonals of a 32 x 32 tile: sums dS over each (one lane a diagonal) and adds them to `sums`.
// Distances at or past max_distance share a bucket with everything further and go to the lane's two registers.
struct BiasGrad {
  static constexpr int LD = 36;  // floats: keeps the four-word writes aligned, neighbouring lanes of a diagonal read stay apart
  float below = 0.f, above = 0.f;
  __device__ __forceinline__ void add(const float (&ds)[16], int rel0 /* key0 - pos0 */, int md, float* scratch, float* sums, int lane) {
    const int half = lane >> 5, col = lane & 31;
    if (rel0 + 31 <= -md || rel0 - 31 >= md) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) x += ds[i];
      if (rel0 < 0) below += x;
      else above += x;
      return;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(scratch + col * LD + 8 * g + 4 * half) = f32x4{ds[4 * g], ds[4 * g + 1], ds[4 * g + 2], ds[4 * g + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float x = 0.f;
    const int d = lane - 31;  // key - query within the tile; lane 63 has none
#pragma unroll
    for (int qq = 0; qq < 32; ++qq) {
      const int kk = d + qq;
      const float v = scratch[qq * LD + (kk & 31)];
      x += (kk >= 0 && kk < 32) ? v : 0.f;
    }
    if (lane == 63) return;
    const int rel = rel0 + d;
    if (rel <= -md) below += x;
    else if (rel >= md) above += x;
    else sums[rel + md] += x;
  }
};

// Shapes of a workgroup, as in the forward pass: wide = 4 waves of 32 stationary rows each against every subtile of a tile; narrow = 32
// stationary rows, the waves on different subtiles, joined at the end.
template <class T, int DP, bool WIDE>
struct BackwardShape {
  static constexpr int NP = Type<T>::NP;
  static constexpr int WS = WIDE ? 4 : 1, WM = WIDE ? 1 : NP == 1 ? (DP == 256 ? 2 : 4) : DP == 64 ? 4 : DP == 128 ? 2 : 1;
  static constexpr int NS = WIDE && NP == 1 && DP < 256 ? 2 : 1;  // subtiles of a tile per wave
  static constexpr int WAVES = WS * WM, THREADS = 64 * WAVES, BM = 32 * WM * NS;
  static constexpr int BUFS = WIDE && !(NP == 3 && DP == 256) ? 2 : 1;  // two where they leave room for the position bias's tables
  static constexpr bool AHEAD = WIDE || DP * NP <= 256;                 // the next tile is requested before this one's arithmetic
  static constexpr bool EARLY = NP == 3 && BUFS == 2;                   // it goes to LDS beside the arithmetic (forward pass)
  static constexpr bool RAW = NP == 3 && DP == 256;
  // output columns of a workgroup: both sums and both stationary operands have to fit the registers
  static constexpr int DA = DP > 128 ? 128 : DP, PARTS = DP / DA, DT = DA / 32;
  using TL = Tile<T, DP, BM>;
  static constexpr size_t TILES = 2 * BUFS * TL::BYTES, SUMS = WM > 1 ? (size_t)WM * 32 * (DA + 4) * 4 : 0;
  static constexpr size_t BODY = TILES > SUMS ? TILES : SUMS;
  static constexpr int DQ_WAVES = DP * NP <= 64 ? 2 : 1, DKV_WAVES = DP * NP <= 64 ? 2 : 1;  // per SIMD
};

// Sum over the waves of the narrow shape, through LDS in the tiles' place, and out: row of column c = base + c * stride.
template <class S, class T>
__device__ __forceinline__ void join_and_store(const f32x16 (&acc)[S::DT], float* sums, T* base, int64_t stride, int rows, int d0, int D,
                                               float scale, int wave, int lane, int tid) {
  constexpr int LD = S::DA + 4, TPC = S::THREADS / 32;
  const int half = lane >> 5, col = lane & 31;
  __syncthreads();
#pragma unroll
  for (int dt = 0; dt < S::DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(sums + (wave * 32 + col) * LD + dt * 32 + 8 * g + 4 * half) =
          f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
  __syncthreads();
  const int c = tid / TPC;
  if (c < rows) {
    T* row = base + c * stride;
#pragma unroll
    for (int d = (tid % TPC) * 4; d < S::DA; d += TPC * 4) {
      f32x4 x = *reinterpret_cast<const f32x4*>(sums + c * LD + d);
#pragma unroll
      for (int w = 1; w < S::WM; ++w) x += *reinterpret_cast<const f32x4*>(sums + (w * 32 + c) * LD + d);
      store4<T>(row, d0 + d, D, x[0] * scale, x[1] * scale, x[2] * scale, x[3] * scale);
    }
  }
}
template <class S, class T>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[S::DT], T* row, int d0, int D, float scale, int half) {
#pragma unroll
  for (int dt = 0; dt < S::DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4<T>(row, d0 + dt * 32 + 8 * g + 4 * half, D, acc[dt][4 * g] * scale, acc[dt][4 * g + 1] * scale, acc[dt][4 * g + 2] * scale,
                acc[dt][4 * g + 3] * scale);
}

// dq (and with BIAS == 2 the table's gradient): queries stationary, key tiles through LDS.
//
// delta = rowsum(dout * out) serves a softmax gradient well as long as out is exact; in bfloat16 it carries out's rounding, and a bucket that
// holds most of a row's keys adds that error up over all rows.  There the table's gradient takes delta = sum_j P dP from a first walk over the
// keys instead.
template <class T, int DP, int BIAS, bool WIDE>
__global__ __launch_bounds__((BackwardShape<T, DP, WIDE>::THREADS), (BackwardShape<T, DP, WIDE>::DQ_WAVES)) void attention_dq_kernel(Params p) {
  using S = BackwardShape<T, DP, WIDE>;
  using TL = typename S::TL;
  constexpr int BN = S::BM, NC2 = DP / 16, BUFS = S::BUFS, NT = S::THREADS;
  constexpr bool TWICE = BIAS == 2 && sizeof(T) == 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* kt = smem;
  char* vt = smem + BUFS * TL::BYTES;
  float* wave_delta = reinterpret_cast<float*>(smem + S::BODY);  // [WM][32]
  int* word = reinterpret_cast<int*>(wave_delta + 4 * 32);
  float* lut = reinterpret_cast<float*>(word + 4);
  const int lut_len = BIAS ? 2 * p.max_distance + 1 : 0, lut_pad = (lut_len + 3) & ~3;
  float* scratch = lut + lut_pad;                        // [WAVES][32 * LD]
  float* sums = scratch + S::WAVES * 32 * BiasGrad::LD;  // [WAVES][lut_pad]
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ws = WIDE ? wave : 0, wm = WIDE ? 0 : wave;
  const int nt = (p.Tq + 32 * S::WS - 1) / (32 * S::WS), n = p.B * p.H * nt * S::PARTS;
  int item = xcd_item(n);
  if (item >= n) return;
  const int d0 = (item % S::PARTS) * S::DA;
  item /= S::PARTS;
  const int bh = item / nt, b = bh / p.H, h = bh - b * p.H, qt = p.causal ? nt - 1 - item % nt : item % nt;
  const int q0 = qt * 32 * S::WS + 32 * ws;
  const int off = start_of(p, b), kvh = h / p.group;
  const T* kb = reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h;
  const T* vb = reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h;
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  const int qi = q0 + col, qc = min(qi, p.Tq - 1), pos = qi + off;
  const int pos_lo = q0 + off, pos_hi = pos_lo + 31;
  Stationary<T, DP, S::RAW> q, go;
  float delta = 0.f;
  {
    const T* gr = reinterpret_cast<const T*>(p.dout) + b * p.do_b + h * p.do_h + qc * p.do_t;
    q.load(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h + qc * p.q_t, half, p.D, true);
    go.load(gr, half, p.D, true);
    if (!TWICE) {
      const T* orow = reinterpret_cast<const T*>(p.o_in) + b * p.oi_b + h * p.oi_h + qc * p.oi_t;
#pragma unroll
      for (int c = 0; c < NC2; ++c) {
        const Raw<T> g = load_chunk<T>(gr, 2 * c + half, p.D), o = load_chunk<T>(orow, 2 * c + half, p.D);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta += (float)g.x[e] * (float)o.x[e];
      }
      delta = both_sum(delta);
    }
  }
  const float lse = qi < p.Tq ? p.lse[(int64_t)bh * p.Tq + qi] : -INFINITY;
  const float lse2 = lse == -INFINITY ? INFINITY : lse * kLog2e;  // a row without keys, or none at all: P = exp2(.. - inf) = 0
  if constexpr (BIAS != 0) fill_lut(p, h, lut, tid, NT);
  if constexpr (BIAS == 2)
    for (int i = tid; i < S::WAVES * lut_pad; i += NT) sums[i] = 0.f;
  const int end = key_end(p, b, min(qt * 32 * S::WS + 32 * S::WS - 1, p.Tq - 1) + off, word, tid, NT);
  const int tiles = (end + BN - 1) / BN;
  f32x16 acc[S::DT] = {};
  BiasGrad bias_grad;
  Stage<T, DP, BN, NT> sk, sv;
  sk.start(kb, p.k_t, end, p.D, tid);
  sv.start(vb, p.v_t, end, p.D, tid);
  auto load = [&](int t, const RowBits& use) {
    sk.load(t * BN, mask ? &use : nullptr, tid);
    sv.load(t * BN, mask ? &use : nullptr, tid);
  };
  auto store = [&](int t) {
    const int o = t & (BUFS - 1);
    sk.store(kt + o * TL::BYTES, tid);
    sv.store(vt + o * TL::BYTES, tid);
  };
#pragma unroll
  for (int walk = TWICE ? 0 : 1; walk < 2; ++walk) {
    // the order of a round: as in the forward pass
    KeyBits<BN> keys(mask, end, lane, 0);
    RowBits use = keys.next(0), use1 = keys.next(BN), use2;  // of tiles t, t + 1, t + 2
    load(0, use);
    store(0);
    if (S::EARLY) load(1, use1);
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
      const char *kk = kt + (t & (BUFS - 1)) * TL::BYTES, *vv = vt + (t & (BUFS - 1)) * TL::BYTES;
      use2 = keys.next((t + 2) * BN);
      if (!S::EARLY && S::AHEAD) load(t + 1, use1);
#pragma unroll
      for (int x = 0; x < S::NS; ++x) {
        const int sub = S::NS * wm + x, key0 = t * BN + sub * 32;
        const bool work = key0 < end && !(p.causal && key0 > pos_hi);
        f32x16 raw = {}, dp = {};
        if (work) {
#pragma unroll
          for (int c = 0; c < NC2; ++c)
            mma2(TL::row_chunk(kk, sub * 32 + col, 2 * c + half), q.get(c), raw, TL::row_chunk(vv, sub * 32 + col, 2 * c + half), go.get(c), dp,
                 [](int) {});
        }
        if (x == 0 && S::EARLY) {
          store(t + 1);
          load(t + 2, use2);
        }
        if (work) {
          float pr[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pr[i] = raw[i];
          finish_scores<BIAS != 0>(p, pr, key0, pos, pos_lo, pos_hi, use.of(sub), lut, half);
#pragma unroll
          for (int i = 0; i < 16; ++i) pr[i] = __builtin_amdgcn_exp2f(pr[i] - lse2);
          if (TWICE && walk == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) delta += pr[i] * dp[i];
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) pr[i] *= dp[i] - delta;
            if constexpr (BIAS == 2)
              if (d0 == 0) bias_grad.add(pr, key0 - pos_lo, p.max_distance, scratch + wave * 32 * BiasGrad::LD, sums + wave * lut_pad, lane);
            column_product<T, TL>(kk, sub * 32, d0, Weights<T>(pr), acc, lane);
          }
        }
      }
      if (!S::EARLY) {
        if (BUFS == 1) __syncthreads();
        if (!S::AHEAD) load(t + 1, use1);
        store(t + 1);
      }
      use = use1;
      use1 = use2;
      __syncthreads();
    }
    if (TWICE && walk == 0) {
      delta = both_sum(delta);
      if constexpr (S::WM > 1) {
        if (half == 0) wave_delta[wm * 32 + col] = delta;
        __syncthreads();
        delta = 0.f;
#pragma unroll
        for (int w = 0; w < S::WM; ++w) delta += wave_delta[w * 32 + col];
      }
    }
  }
  if (half == 0 && wm == 0 && d0 == 0 && qi < p.Tq) p.delta[(int64_t)bh * p.Tq + qi] = delta;
  T* out = reinterpret_cast<T*>(p.dq) + b * p.dq_b + h * p.dq_h;
  if constexpr (S::WM > 1)
    join_and_store<S>(acc, reinterpret_cast<float*>(smem), out + q0 * p.dq_t, p.dq_t, p.Tq - q0, d0, p.D, p.scale, wave, lane, tid);
  else if (qi < p.Tq)
    store_rows<S>(acc, out + qi * p.dq_t, d0, p.D, p.scale, half);
  if constexpr (BIAS == 2) {
    if (d0 != 0) return;
    for (int m = 1; m < 64; m <<= 1) {
      bias_grad.below += __shfl_xor(bias_grad.below, m);
      bias_grad.above += __shfl_xor(bias_grad.above, m);
    }
    if (lane == 0) {
      sums[wave * lut_pad] = bias_grad.below;
      sums[wave * lut_pad + 2 * p.max_distance] = bias_grad.above;
    }
    __syncthreads();
    // the waves' sums, then a bucket's distances, each in a fixed order
    for (int i = tid; i < lut_len; i += NT) {
      float x = sums[i];
      for (int w = 1; w < S::WAVES; ++w) x += sums[w * lut_pad + i];
      sums[i] = x;
    }
    __syncthreads();
    for (int i = tid; i < p.buckets; i += NT) p.dtable_part[((int64_t)(b * nt + qt) * p.H + h) * p.buckets + i] = bucket_sum(p, sums, i);
  }
}

// dk, dv: keys of one key head stationary; tiles of queries and their output gradients through LDS, over all heads of the group.
template <class T, int DP, bool BIAS, bool WIDE>
__global__ __launch_bounds__((BackwardShape<T, DP, WIDE>::THREADS), (BackwardShape<T, DP, WIDE>::DKV_WAVES)) void attention_dkv_kernel(Params p) {
  using S = BackwardShape<T, DP, WIDE>;
  using TL = typename S::TL;
  constexpr int BM = S::BM, NC2 = DP / 16, BUFS = S::BUFS, NT = S::THREADS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* qt = smem;
  char* gt = smem + BUFS * TL::BYTES;
  float* stat = reinterpret_cast<float*>(smem + S::BODY);  // [BUFS][2][BM]: lse in log2 units, delta
  float* lut = stat + BUFS * 2 * BM;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ws = WIDE ? wave : 0, wm = WIDE ? 0 : wave;
  const int nt = (p.Tk + 32 * S::WS - 1) / (32 * S::WS), n = p.B * p.Hkv * nt * S::PARTS;
  int item = xcd_item(n);
  if (item >= n) return;
  const int d0 = (item % S::PARTS) * S::DA;
  item /= S::PARTS;
  const int bh = item / nt, b = bh / p.Hkv, kvh = bh - b * p.Hkv, k0 = (item % nt) * 32 * S::WS, kw = k0 + 32 * ws;
  const int off = start_of(p, b), key = kw + col, kc = min(key, p.Tk - 1);
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  int end = p.Tk;
  if (p.key_lens) end = min(end, max(p.key_lens[b], 0));
  if (p.causal) end = min(end, max(p.Tq + off, 0));  // past the last query's reach
  const bool ok = key < end && !(mask && mask[kc]);
  Stationary<T, DP, S::RAW> k, v;
  k.load(reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h + kc * p.k_t, half, p.D, ok);
  v.load(reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h + kc * p.v_t, half, p.D, ok);
  const float add = ok ? 0.f : -INFINITY;
  f32x16 dk[S::DT] = {}, dv[S::DT] = {};
  // under causality queries before key - off see nothing of this block
  const int qt_n = (p.Tq + BM - 1) / BM, qt_0 = p.causal ? min(max(k0 - off, 0) / BM, qt_n) : 0, per = qt_n - qt_0;
  const int steps = k0 < end ? per * p.group : 0;
  Stage<T, DP, BM, NT> sq, sg;
  sq.start(nullptr, p.q_t, p.Tq, p.D, tid);
  sg.start(nullptr, p.do_t, p.Tq, p.D, tid);
  float s_lse = 0.f, s_delta = 0.f;
  auto load = [&](int it) {
    if (it >= steps) return;
    const int h = kvh * p.group + it / per, r0 = (qt_0 + it % per) * BM;
    sq.base = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h);
    sg.base = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.dout) + b * p.do_b + h * p.do_h);
    sq.load(r0, nullptr, tid);
    sg.load(r0, nullptr, tid);
    if (tid < BM) {
      const int64_t row = ((int64_t)b * p.H + h) * p.Tq + r0 + tid;
      const float l = r0 + tid < p.Tq ? p.lse[row] : -INFINITY;
      s_lse = l == -INFINITY ? INFINITY : l * kLog2e;
      s_delta = r0 + tid < p.Tq ? p.delta[row] : 0.f;
    }
  };
  auto store = [&](int it) {
    const int o = it & (BUFS - 1);
    sq.store(qt + o * TL::BYTES, tid);
    sg.store(gt + o * TL::BYTES, tid);
    if (tid < BM) {
      stat[o * 2 * BM + tid] = s_lse;
      stat[(o * 2 + 1) * BM + tid] = s_delta;
    }
  };
  load(0);
  store(0);
  if (S::EARLY) load(1);
  __syncthreads();
  for (int it = 0; it < steps; ++it) {
    if constexpr (BIAS) {
      if (it % per == 0) {
        fill_lut(p, kvh * p.group + it / per, lut, tid, NT);
        __syncthreads();
      }
    }
    const int o = it & (BUFS - 1), r0 = (qt_0 + it % per) * BM;
    const char *qq = qt + o * TL::BYTES, *gg = gt + o * TL::BYTES;
    if (!S::EARLY && S::AHEAD) load(it + 1);
#pragma unroll
    for (int x = 0; x < S::NS; ++x) {
      const int sub = S::NS * wm + x, i0 = r0 + sub * 32, p0 = i0 + off;  // position of the subtile's first query
      const bool work = kw < end && i0 < p.Tq && !(p.causal && kw > p0 + 31);
      f32x16 raw = {}, dp = {};
      if (work) {
#pragma unroll
        for (int c = 0; c < NC2; ++c)
          mma2(TL::row_chunk(qq, sub * 32 + col, 2 * c + half), k.get(c), raw, TL::row_chunk(gg, sub * 32 + col, 2 * c + half), v.get(c), dp,
               [](int) {});
      }
      if (x == 0 && S::EARLY) {
        store(it + 1);
        load(it + 2);
      }
      if (work) {
        float s[16];
        if constexpr (BIAS) {
          const int md = p.max_distance;
          if (kw + 31 - p0 <= -md || kw - (p0 + 31) >= md) {
            const float far = lut[kw > p0 ? 2 * md : 0] + add;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = fmaf(raw[i], p.scale2, far);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = fmaf(raw[i], p.scale2, lut[min(max(key - p0 - moving_row(i, half), -md), md) + md] + add);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = fmaf(raw[i], p.scale2, add);
        }
        if (p.causal && kw + 31 > p0) {
          const int first = key - p0 - 4 * half;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = first > moving_row(i, 0) ? -INFINITY : s[i];
        }
        const float* l2 = stat + o * 2 * BM + sub * 32 + 4 * half;
        float ds[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 l = *reinterpret_cast<const f32x4*>(l2 + 8 * g), de = *reinterpret_cast<const f32x4*>(l2 + BM + 8 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * g + e;
            s[i] = __builtin_amdgcn_exp2f(s[i] - l[e]);
            ds[i] = s[i] * (dp[i] - de[e]);
          }
        }
        column_product<T, TL>(gg, sub * 32, d0, Weights<T>(s), dv, lane);
        column_product<T, TL>(qq, sub * 32, d0, Weights<T>(ds), dk, lane);
      }
    }
    if (!S::EARLY) {
      if (BUFS == 1) __syncthreads();
      if (!S::AHEAD) load(it + 1);
      store(it + 1);
    }
    __syncthreads();
  }
  T* kout = reinterpret_cast<T*>(p.dk) + b * p.dk_b + kvh * p.dk_h;
  T* vout = reinterpret_cast<T*>(p.dv) + b * p.dv_b + kvh * p.dv_h;
  if constexpr (S::WM > 1) {
    float* sums = reinterpret_cast<float*>(smem);
    join_and_store<S>(dk, sums, kout + kw * p.dk_t, p.dk_t, p.Tk - kw, d0, p.D, p.scale, wave, lane, tid);
    join_and_store<S>(dv, sums, vout + kw * p.dv_t, p.dv_t, p.Tk - kw, d0, p.D, 1.f, wave, lane, tid);
  } else if (key < p.Tk) {
    store_rows<S>(dk, kout + key * p.dk_t, d0, p.D, p.scale, half);
    store_rows<S>(dv, vout + key * p.dv_t, d0, p.D, 1.f, half);
  }
}

// ------------------------------------------------------------------ host

template <class T, int DP, int BIAS, bool WIDE>
static int launch_dq(const Params& p, hipStream_t st) {
  using S = BackwardShape<T, DP, WIDE>;
  static std::atomic<uint64_t> done{0};
  const size_t lut = BIAS ? (size_t)(2 * p.max_distance + 4) * 4 : 0;
  return launch(&attention_dq_kernel<T, DP, BIAS, WIDE>, &done, (int64_t)p.B * p.H * ((p.Tq + 32 * S::WS - 1) / (32 * S::WS)) * S::PARTS, S::THREADS,
                S::BODY + 4 * 32 * 4 + 16 + lut + (BIAS == 2 ? S::WAVES * (32 * BiasGrad::LD * 4 + lut) : 0), p, st);
}
template <class T, int DP, bool BIAS, bool WIDE>
static int launch_dkv(const Params& p, hipStream_t st) {
  using S = BackwardShape<T, DP, WIDE>;
  static std::atomic<uint64_t> done{0};
  const size_t lut = BIAS ? (size_t)(2 * p.max_distance + 4) * 4 : 0;
  return launch(&attention_dkv_kernel<T, DP, BIAS, WIDE>, &done, (int64_t)p.B * p.Hkv * ((p.Tk + 32 * S::WS - 1) / (32 * S::WS)) * S::PARTS,
                S::THREADS, S::BODY + S::BUFS * 2 * S::BM * 4 + lut, p, st);
}

template <class T, int DP, int BIAS>
static int launch_backward(const Params& p, float* dtable, hipStream_t st) {
  if (p.wide_dq ? launch_dq<T, DP, BIAS, true>(p, st) : launch_dq<T, DP, BIAS, false>(p, st)) return 1;
  if (p.dk && p.Tk && (p.wide_dkv ? launch_dkv<T, DP, BIAS != 0, true>(p, st) : launch_dkv<T, DP, BIAS != 0, false>(p, st))) return 1;
  if (BIAS == 2) return launch_table_sum<float>(p.dtable_part, p.B * dq_tiles(p), p.H, p.buckets, dtable, st);
  return 0;
}

template <class T, int DP>
int backward(const Params& p, float* dtable, hipStream_t st) {
  return !p.table ? launch_backward<T, DP, 0>(p, dtable, st) : dtable ? launch_backward<T, DP, 2>(p, dtable, st) : launch_backward<T, DP, 1>(p, dtable, st);
}

}  // namespace attn
}  // namespace wrnn
