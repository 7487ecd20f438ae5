// Self-attention, backward.  With P recomputed from the forward pass's log-sum-exp:
//   dv = P^T dout,  dP = dout v^T,  delta = rowsum(dout * out),  dS = P * (dP - delta),  dq = scale * dS k,  dk = scale * dS^T q,
//   dtable[n, h] = sum of dS over the pairs whose distance falls in bucket n.
//
// Two kernels, each with its own output rows stationary, so that every sum has one owner and one order (no atomics: the same
// inputs give the same bits): dq walks the keys, dk / dv walk the queries of all heads that share them.  Seven tile products
// in place of the five of a form that adds dq up in memory.
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

template <class T, int DP>
constexpr int back_tile() {  // moving rows of a tile in LDS
  return sizeof(T) == 2 && DP < 256 ? 64 : 32;
}
// Two buffers for each tile where they leave room for the position bias's tables.
template <class T, int DP>
constexpr int back_buffers() {
  return sizeof(T) == 4 && DP == 256 ? 1 : 2;
}

// dq (and with BIAS == 2 the table's gradient): 128 queries of one head per workgroup, 32 per wave, key tiles through LDS.
//
// delta = rowsum(dout * out) serves a softmax gradient well as long as out is exact; in bfloat16 it carries out's rounding, and a bucket that
// holds most of a row's keys adds that error up over all rows.  There the table's gradient takes delta = sum_j P dP from a first walk over the
// keys instead.
template <class T, int DP, int BIAS>
__global__ __launch_bounds__(256, DP * Type<T>::NP <= 128 ? 2 : 1) void attention_dq_kernel(Params p) {
  constexpr int BN = back_tile<T, DP>(), NC2 = DP / 16, DA = DP > 128 ? 128 : DP, DT = DA / 32, PARTS = DP / DA, BUFS = back_buffers<T, DP>();
  constexpr bool TWICE = BIAS == 2 && sizeof(T) == 2, RAW = sizeof(T) == 4 && DP == 256;
  using TL = Tile<T, DP, BN>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* kt = smem;
  char* vt = smem + BUFS * TL::BYTES;
  int* word = reinterpret_cast<int*>(smem + 2 * BUFS * TL::BYTES);
  float* lut = reinterpret_cast<float*>(word + 4);
  const int lut_len = BIAS ? 2 * p.max_distance + 1 : 0, lut_pad = (lut_len + 3) & ~3;
  float* scratch = lut + lut_pad;                 // [4][32 * LD]
  float* sums = scratch + 4 * 32 * BiasGrad::LD;  // [4][lut_pad]
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = tid >> 6;
  const int nt = (p.Tq + 127) / 128, n = p.B * p.H * nt * PARTS;
  int item = xcd_item(n);
  if (item >= n) return;
  const int d0 = (item % PARTS) * DA;
  item /= PARTS;
  const int bh = item / nt, b = bh / p.H, h = bh - b * p.H;
  const int q0 = (p.causal ? nt - 1 - item % nt : item % nt) * 128;
  const int off = start_of(p, b), kvh = h / p.group;
  const T* kb = reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h;
  const T* vb = reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h;
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  const int qi = q0 + wave * 32 + (lane & 31), qc = min(qi, p.Tq - 1), pos = qi + off;
  const int pos_lo = q0 + wave * 32 + off, pos_hi = pos_lo + 31;
  Stationary<T, DP, RAW> q, go;
  float delta = 0.f;
  {
    const T* gr = reinterpret_cast<const T*>(p.dout) + b * p.do_b + h * p.do_h + qc * p.do_t;
    q.load(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h + qc * p.q_t, half, p.D, p.vec, true);
    go.load(gr, half, p.D, p.vec, true);
    if (!TWICE) {
      const T* orow = reinterpret_cast<const T*>(p.o_in) + b * p.oi_b + h * p.oi_h + qc * p.oi_t;
#pragma unroll
      for (int c = 0; c < NC2; ++c) {
        const Raw<T> g = load_chunk<T>(gr, 2 * c + half, p.D, p.vec), o = load_chunk<T>(orow, 2 * c + half, p.D, p.vec);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta += (float)g.x[e] * (float)o.x[e];
      }
      delta = both_sum(delta);
    }
  }
  const float lse = qi < p.Tq ? p.lse[(int64_t)bh * p.Tq + qi] : -INFINITY;
  const float lse2 = lse == -INFINITY ? INFINITY : lse * kLog2e;  // a row without keys, or none at all: P = exp2(.. - inf) = 0
  if constexpr (BIAS != 0) fill_lut(p, h, lut, tid, 256);
  if constexpr (BIAS == 2)
    for (int i = tid; i < 4 * lut_pad; i += 256) sums[i] = 0.f;
  const int end = key_end(p, b, min(q0 + 127, p.Tq - 1) + off, word, tid, 256);
  const int tiles = (end + BN - 1) / BN;
  f32x16 acc[DT] = {};
  BiasGrad bias_grad;
  Stage<T, DP, BN> sk, sv;
  KeyBits bits(mask, end, lane);
  auto load = [&](int t) {
    sk.load(kb, p.k_t, t * BN, end, p.D, p.vec, tid);
    sv.load(vb, p.v_t, t * BN, end, p.D, p.vec, tid);
    bits.load(t * BN);
  };
  auto store = [&](int t) {
    const uint64_t use = bits.get(t * BN);
    const int o = t & (BUFS - 1);
    sk.store(kt + o * TL::BYTES, use, tid);
    sv.store(vt + o * TL::BYTES, use, tid);
    return use;
  };
  const bool live = q0 + wave * 32 < p.Tq;
#pragma unroll
  for (int walk = TWICE ? 0 : 1; walk < 2; ++walk) {
    uint64_t use = 0, next = 0;
    if (tiles) {
      load(0);
      use = store(0);
    }
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
      if (t + 1 < tiles) load(t + 1);
      const char *kk = kt + (t & (BUFS - 1)) * TL::BYTES, *vv = vt + (t & (BUFS - 1)) * TL::BYTES;
      if (live) {
#pragma unroll
        for (int sub = 0; sub < BN / 32; ++sub) {
          const int key0 = t * BN + sub * 32;
          if (key0 >= end || (p.causal && key0 > pos_hi)) break;
          f32x16 raw = {}, dp = {};
#pragma unroll
          for (int c = 0; c < NC2; ++c) {
            raw = mma(TL::row_chunk(kk, sub * 32 + (lane & 31), 2 * c + half), q.get(c), raw);
            dp = mma(TL::row_chunk(vv, sub * 32 + (lane & 31), 2 * c + half), go.get(c), dp);
          }
          float pr[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pr[i] = raw[i];
          finish_scores<BIAS != 0>(p, pr, key0, pos, pos_lo, pos_hi, (uint32_t)(use >> (32 * sub)), lut, half);
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
      if (BUFS == 1) __syncthreads();
      if (t + 1 < tiles) next = store(t + 1);
      use = next;
      __syncthreads();
    }
    if (TWICE && walk == 0) delta = both_sum(delta);
  }
  if (qi < p.Tq) {
    T* row = reinterpret_cast<T*>(p.dq) + b * p.dq_b + h * p.dq_h + qi * p.dq_t;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        store4<T>(row, d0 + dt * 32 + 8 * g + 4 * half, p.D, p.vec, acc[dt][4 * g] * p.scale, acc[dt][4 * g + 1] * p.scale,
                  acc[dt][4 * g + 2] * p.scale, acc[dt][4 * g + 3] * p.scale);
    if (half == 0 && d0 == 0) p.delta[(int64_t)bh * p.Tq + qi] = delta;
  }
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
    // the four waves' sums, then a bucket's distances, each in a fixed order
    for (int i = tid; i < lut_len; i += 256) {
      float x = sums[i];
      for (int w = 1; w < 4; ++w) x += sums[w * lut_pad + i];
      sums[i] = x;
    }
    __syncthreads();
    if (tid < p.buckets) {
      const int64_t row = (int64_t)(b * nt + q0 / 128) * p.H + h;
      p.dtable_part[row * p.buckets + tid] = bucket_sum(p, sums, tid);
    }
  }
}

// dk, dv: 128 keys of one key head per workgroup, 32 per wave; tiles of queries and their output gradients through LDS, over all heads of
// the group.
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(256, DP * Type<T>::NP <= 64 ? 2 : 1) void attention_dkv_kernel(Params p) {
  constexpr int BM = back_tile<T, DP>(), NC2 = DP / 16, DA = DP > 128 ? 128 : DP, DT = DA / 32, PARTS = DP / DA, BUFS = back_buffers<T, DP>();
  constexpr bool RAW = sizeof(T) == 4 && DP == 256;
  using TL = Tile<T, DP, BM>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* qt = smem;
  char* gt = smem + BUFS * TL::BYTES;
  float* stat = reinterpret_cast<float*>(smem + 2 * BUFS * TL::BYTES);  // [BUFS][2][BM]: lse in log2 units, delta
  float* lut = stat + 4 * BM;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = tid >> 6;
  const int nt = (p.Tk + 127) / 128, n = p.B * p.Hkv * nt * PARTS;
  int item = xcd_item(n);
  if (item >= n) return;
  const int d0 = (item % PARTS) * DA;
  item /= PARTS;
  const int bh = item / nt, b = bh / p.Hkv, kvh = bh - b * p.Hkv, k0 = (item % nt) * 128;
  const int off = start_of(p, b), key = k0 + wave * 32 + (lane & 31), kc = min(key, p.Tk - 1), kw = k0 + wave * 32;
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  int end = p.Tk;
  if (p.key_lens) end = min(end, max(p.key_lens[b], 0));
  if (p.causal) end = min(end, max(p.Tq + off, 0));  // past the last query's reach
  const bool ok = key < end && !(mask && mask[kc]);
  Stationary<T, DP, RAW> k, v;
  k.load(reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h + kc * p.k_t, half, p.D, p.vec, ok);
  v.load(reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h + kc * p.v_t, half, p.D, p.vec, ok);
  const float add = ok ? 0.f : -INFINITY;
  f32x16 dk[DT] = {}, dv[DT] = {};
  // under causality queries before key - off see nothing of this block
  const int qt_n = (p.Tq + BM - 1) / BM, qt_0 = p.causal ? min(max(k0 - off, 0) / BM, qt_n) : 0, per = qt_n - qt_0;
  const int steps = k0 < end ? per * p.group : 0;
  Stage<T, DP, BM> sq, sg;
  float s_lse = 0.f, s_delta = 0.f;
  auto load = [&](int it) {
    const int h = kvh * p.group + it / per, r0 = (qt_0 + it % per) * BM;
    sq.load(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h, p.q_t, r0, p.Tq, p.D, p.vec, tid);
    sg.load(reinterpret_cast<const T*>(p.dout) + b * p.do_b + h * p.do_h, p.do_t, r0, p.Tq, p.D, p.vec, tid);
    if (tid < BM) {
      const int64_t row = ((int64_t)b * p.H + h) * p.Tq + r0 + tid;
      const float l = r0 + tid < p.Tq ? p.lse[row] : -INFINITY;
      s_lse = l == -INFINITY ? INFINITY : l * kLog2e;
      s_delta = r0 + tid < p.Tq ? p.delta[row] : 0.f;
    }
  };
  auto store = [&](int it) {
    const int o = it & (BUFS - 1);
    sq.store(qt + o * TL::BYTES, ~0ull, tid);
    sg.store(gt + o * TL::BYTES, ~0ull, tid);
    if (tid < BM) {
      stat[o * 2 * BM + tid] = s_lse;
      stat[(o * 2 + 1) * BM + tid] = s_delta;
    }
  };
  if (steps) {
    load(0);
    store(0);
  }
  for (int it = 0; it < steps; ++it) {
    if constexpr (BIAS) {
      if (it % per == 0) {
        __syncthreads();
        fill_lut(p, kvh * p.group + it / per, lut, tid, 256);
      }
    }
    __syncthreads();
    if (it + 1 < steps) load(it + 1);
    const int o = it & (BUFS - 1), r0 = (qt_0 + it % per) * BM;
    const char *qq = qt + o * TL::BYTES, *gg = gt + o * TL::BYTES;
    if (kw < end) {
#pragma unroll
      for (int sub = 0; sub < BM / 32; ++sub) {
        const int i0 = r0 + sub * 32, p0 = i0 + off;  // position of the subtile's first query
        if (i0 >= p.Tq) break;
        if (p.causal && kw > p0 + 31) continue;
        f32x16 raw = {}, dp = {};
#pragma unroll
        for (int c = 0; c < NC2; ++c) {
          raw = mma(TL::row_chunk(qq, sub * 32 + (lane & 31), 2 * c + half), k.get(c), raw);
          dp = mma(TL::row_chunk(gg, sub * 32 + (lane & 31), 2 * c + half), v.get(c), dp);
        }
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
    if (BUFS == 1) __syncthreads();
    if (it + 1 < steps) store(it + 1);
  }
  if (key >= p.Tk) return;
  T* kr = reinterpret_cast<T*>(p.dk) + b * p.dk_b + kvh * p.dk_h + key * p.dk_t;
  T* vr = reinterpret_cast<T*>(p.dv) + b * p.dv_b + kvh * p.dv_h + key * p.dv_t;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = d0 + dt * 32 + 8 * g + 4 * half;
      store4<T>(kr, d, p.D, p.vec, dk[dt][4 * g] * p.scale, dk[dt][4 * g + 1] * p.scale, dk[dt][4 * g + 2] * p.scale, dk[dt][4 * g + 3] * p.scale);
      store4<T>(vr, d, p.D, p.vec, dv[dt][4 * g], dv[dt][4 * g + 1], dv[dt][4 * g + 2], dv[dt][4 * g + 3]);
    }
}

// ------------------------------------------------------------------ host

static size_t aligned(size_t x) { return (x + 255) & ~size_t(255); }
static size_t delta_bytes(const Params& p) { return aligned((size_t)p.B * p.H * p.Tq * sizeof(float)); }
static int dtable_rows(const Params& p) { return p.B * ((p.Tq + 127) / 128); }

template <class T, int DP, int BIAS>
static int launch_backward(const Params& p, float* dtable, hipStream_t st) {
  constexpr int PARTS = DP > 128 ? 2 : 1;
  constexpr size_t tiles = 2 * back_buffers<T, DP>() * Tile<T, DP, back_tile<T, DP>()>::BYTES;
  const size_t lut = BIAS ? (size_t)(2 * p.max_distance + 4) * 4 : 0;
  static std::atomic<uint64_t> dq_done{0}, dkv_done{0};
  if (launch(&attention_dq_kernel<T, DP, BIAS>, &dq_done, (int64_t)p.B * p.H * ((p.Tq + 127) / 128) * PARTS,
             tiles + 16 + lut + (BIAS == 2 ? 4 * (32 * BiasGrad::LD * 4 + lut) : 0), p, st))
    return 1;
  if (p.dk && p.Tk && launch(&attention_dkv_kernel<T, DP, BIAS != 0>, &dkv_done, (int64_t)p.B * p.Hkv * ((p.Tk + 127) / 128) * PARTS,
                             tiles + 4 * back_tile<T, DP>() * 4 + lut, p, st))
    return 1;
  if (BIAS == 2) {
    return launch_table_sum<float>(p.dtable_part, dtable_rows(p), p.H, p.buckets, dtable, st);
  }
  return 0;
}

template <class T, int DP>
static int launch_bias(const Params& p, float* dtable, hipStream_t st) {
  return !p.table ? launch_backward<T, DP, 0>(p, dtable, st) : dtable ? launch_backward<T, DP, 2>(p, dtable, st) : launch_backward<T, DP, 1>(p, dtable, st);
}

template <class T>
static int launch_dim(const Params& p, float* dtable, hipStream_t st) {
  return p.D <= 64 ? launch_bias<T, 64>(p, dtable, st) : p.D <= 128 ? launch_bias<T, 128>(p, dtable, st) : launch_bias<T, 256>(p, dtable, st);
}

}  // namespace attn
}  // namespace wrnn

using namespace wrnn;

extern "C" size_t wrnn_attention_backward_workspace_bytes(const wrnn_attention_desc* desc) {
  attn::Params p;
  if (attention_params(desc, &p, "wrnn_attention_backward_workspace_bytes") || !p.B || !p.H || !p.Tq) return 0;
  return attn::delta_bytes(p) + (p.table ? attn::aligned((size_t)attn::dtable_rows(p) * p.H * p.buckets * sizeof(float)) : 0);
}

extern "C" int wrnn_attention_backward(const wrnn_attention_desc* desc, const wrnn_attention_grads* g, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  attn::Params p;
  if (attention_params(desc, &p, "wrnn_attention_backward")) return 1;
  WRNN_REQUIRE(g, "wrnn_attention_backward: null gradients");
  if (!p.B || !p.H || !p.Tq) {
    WRNN_REQUIRE(!p.B || !p.H || !p.Tk, "wrnn_attention_backward: no queries; dk, dv and the table's gradient are zero and left to the caller");
    return 0;
  }
  WRNN_REQUIRE(g->out && g->lse && g->dout && g->dq && !g->dk == !g->dv, "wrnn_attention_backward: null pointer");
  WRNN_REQUIRE(!g->dtable || p.table, "wrnn_attention_backward: a table's gradient without a table");
  const size_t need = wrnn_attention_backward_workspace_bytes(desc);
  WRNN_REQUIRE(workspace && workspace_bytes >= need, "wrnn_attention_backward: workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  const int es = desc->dtype == WRNN_FLOAT32 ? 4 : 2;
  auto on16 = [&](const void* x, const int64_t* st) { return attn::rows_on_16(x, st[0], st[1], st[2], es); };
  p.vec = p.vec && on16(g->out, g->out_stride) && on16(g->dout, g->dout_stride) && on16(g->dq, g->dq_stride) &&
          on16(g->dk, g->dk_stride) && on16(g->dv, g->dv_stride);
  for (const int64_t* x : {g->out_stride, g->dout_stride, g->dq_stride, g->dk_stride, g->dv_stride})
    WRNN_REQUIRE(x[2] > -attn::kMaxRowStride && x[2] < attn::kMaxRowStride, "wrnn_attention_backward: position strides are below 2^26 elements");
  p.o_in = g->out, p.oi_b = g->out_stride[0], p.oi_h = g->out_stride[1], p.oi_t = g->out_stride[2];
  p.dout = g->dout, p.do_b = g->dout_stride[0], p.do_h = g->dout_stride[1], p.do_t = g->dout_stride[2];
  p.dq = g->dq, p.dq_b = g->dq_stride[0], p.dq_h = g->dq_stride[1], p.dq_t = g->dq_stride[2];
  p.dk = g->dk, p.dk_b = g->dk_stride[0], p.dk_h = g->dk_stride[1], p.dk_t = g->dk_stride[2];
  p.dv = g->dv, p.dv_b = g->dv_stride[0], p.dv_h = g->dv_stride[1], p.dv_t = g->dv_stride[2];
  p.lse = const_cast<float*>(g->lse);
  p.delta = static_cast<float*>(workspace);
  p.dtable_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + attn::delta_bytes(p));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return desc->dtype == WRNN_FLOAT32 ? attn::launch_dim<float>(p, g->dtable, st) : attn::launch_dim<__bf16>(p, g->dtable, st);
}
