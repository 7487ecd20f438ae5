// Self-attention, forward:  out = softmax(scale * q k^T + bias) v  over the keys that lengths, mask and causality leave.
//
// One pass over the keys with a running maximum and sum per query (kept in 32 bits, in units of log2 so that the exponential is
// one v_exp_f32).  The [Tq, Tk] scores only ever exist as 32 x 32 tiles in registers (attention_tile.h).
#include "attention_tile.h"

namespace wrnn {
namespace attn {

// Running softmax of one query per lane: maximum, sum (this half-wave's share), and the accumulators it scales.
// The maximum only moves when a score exceeds it by more than 8 (a factor 256, far inside float's range): most tiles rescale nothing.
struct Running {
  float m = -3e38f, l = 0.f;
  template <int NS, int DT>
  __device__ __forceinline__ void step(float (&s)[NS][16], f32x16 (&acc)[DT]) {
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
    mx = both_max(mx);
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx), a = exp2f(m - mn);
      m = mn;
      l *= a;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= a;
    }
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[n][i] = __builtin_amdgcn_exp2f(s[n][i] - m);
        l += s[n][i];
      }
  }
};

// Keys of a tile in LDS.
template <class T>
constexpr int key_tile() {
  return sizeof(T) == 2 ? 64 : 32;
}
// Two buffers for each tile where they fit.
template <class T, int DP>
constexpr int forward_buffers() {
  return sizeof(T) == 4 && DP == 256 ? 1 : 2;
}

// 128 queries of one head per workgroup, 32 per wave, against key tiles shared through LDS (two buffers, one barrier a tile).
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(256, DP * Type<T>::NP <= 192 ? 2 : 1) void attention_forward_kernel(Params p) {
  constexpr int BN = key_tile<T>(), NS = BN / 32, NC2 = DP / 16, DT = DP / 32, BUFS = forward_buffers<T, DP>();
  using TL = Tile<T, DP, BN>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* kt = smem;
  char* vt = smem + BUFS * TL::BYTES;
  int* word = reinterpret_cast<int*>(smem + 2 * BUFS * TL::BYTES);
  float* lut = reinterpret_cast<float*>(word + 4);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = tid >> 6;
  const int nt = (p.Tq + 127) / 128, n = p.B * p.H * nt, item = xcd_item(n);
  if (item >= n) return;
  const int bh = item / nt, b = bh / p.H, h = bh - b * p.H;
  const int q0 = (p.causal ? nt - 1 - item % nt : item % nt) * 128;  // under causality the long rows start first
  const int off = start_of(p, b), kvh = h / p.group;
  const T* kb = reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h;
  const T* vb = reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h;
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  const int qi = q0 + wave * 32 + (lane & 31), pos = qi + off;
  const int pos_lo = q0 + wave * 32 + off, pos_hi = pos_lo + 31;
  Stationary<T, DP, false> q;
  q.load(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h + min(qi, p.Tq - 1) * p.q_t, half, p.D, p.vec, true);
  if constexpr (BIAS) fill_lut(p, h, lut, tid, 256);
  const int end = key_end(p, b, min(q0 + 127, p.Tq - 1) + off, word, tid, 256);
  const int tiles = (end + BN - 1) / BN;
  f32x16 acc[DT] = {};
  Running run;
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
  uint64_t use = 0, next = 0;
  if (tiles) {
    load(0);
    use = store(0);
  }
  __syncthreads();
  for (int t = 0; t < tiles; ++t) {
    if (t + 1 < tiles) load(t + 1);
    const char *kk = kt + (t & (BUFS - 1)) * TL::BYTES, *vv = vt + (t & (BUFS - 1)) * TL::BYTES;
    const int key0 = t * BN;
    if (q0 + wave * 32 < p.Tq && !(p.causal && key0 > pos_hi)) {
      f32x16 raw[NS] = {};
#pragma unroll
      for (int c = 0; c < NC2; ++c)
#pragma unroll
        for (int s = 0; s < NS; ++s) raw[s] = mma(TL::row_chunk(kk, s * 32 + (lane & 31), 2 * c + half), q.get(c), raw[s]);
      float s[NS][16];
#pragma unroll
      for (int x = 0; x < NS; ++x) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[x][i] = raw[x][i];
        finish_scores<BIAS>(p, s[x], key0 + 32 * x, pos, pos_lo, pos_hi, (uint32_t)(use >> (32 * x)), lut, half);
      }
      run.step(s, acc);
#pragma unroll
      for (int x = 0; x < NS; ++x) column_product<T, TL>(vv, 32 * x, 0, Weights<T>(s[x]), acc, lane);
    }
    if (BUFS == 1) __syncthreads();
    if (t + 1 < tiles) next = store(t + 1);
    use = next;
    __syncthreads();
  }
  if (qi >= p.Tq) return;
  const float l = both_sum(run.l), inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* orow = reinterpret_cast<T*>(p.out) + b * p.o_b + h * p.o_h + qi * p.o_t;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4<T>(orow, dt * 32 + 8 * g + 4 * half, p.D, p.vec, acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv,
                acc[dt][4 * g + 3] * inv);
  if (half == 0 && p.lse) p.lse[(int64_t)bh * p.Tq + qi] = l == 0.f ? -INFINITY : (run.m + log2f(l)) * kLn2;
}

// Few queries, or too few workgroups of the kernel above: 32 query columns per workgroup (with p.pack the queries of a whole group
// of heads that share k and v), its four waves on different 32-key tiles and further splits of the keys on other workgroups.  A
// wave is on its own until the join: keys go from memory to the matrix instructions' registers, values through a
// private LDS tile of at most 128 columns, both requested one tile ahead where registers allow.
template <class T, int DP>
constexpr int split_columns() {
  return DP > 128 ? 128 : DP;
}
template <class T, int DP>
constexpr size_t split_wave_bytes() {  // a wave's value tile, and later its sums
  const size_t tile = Tile<T, split_columns<T, DP>(), 32>::BYTES, sums = 32 * (DP + 4) * sizeof(float);
  return tile > sums ? tile : sums;
}
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(256, 1) void attention_split_kernel(Params p) {
  constexpr int NC2 = DP / 16, DT = DP / 32, DV = split_columns<T, DP>(), VP = DP / DV, NCV = DV / 8, NV = 32 * NCV / 64;
  constexpr bool AHEAD = DP * sizeof(T) <= 512;
  using TL = Tile<T, DV, 32>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* ml = reinterpret_cast<float*>(smem + 4 * split_wave_bytes<T, DP>());  // [4][2][32]
  int* word = reinterpret_cast<int*>(ml + 4 * 2 * 32);
  float* lut = reinterpret_cast<float*>(word + 4);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = tid >> 6, col = lane & 31;
  char* vt = smem + wave * split_wave_bytes<T, DP>();
  const int heads = p.pack ? p.Hkv : p.H, nq = p.pack ? 1 : (p.Tq + 31) / 32;
  const int n = p.B * heads * nq * p.splits, item = xcd_item(n);
  if (item >= n) return;
  const int split = item % p.splits, r = item / p.splits, qt = r % nq, bh = r / nq, b = bh / heads, hh = bh - b * heads;
  const int lh = p.pack ? col / p.Tq : 0;  // the column's head within the group
  const int h = p.pack ? hh * p.group + min(lh, p.group - 1) : hh, kvh = p.pack ? hh : hh / p.group;
  const int qi = p.pack ? col - lh * p.Tq : qt * 32 + col;
  const int off = start_of(p, b), pos = qi + off;
  const int pos_lo = (p.pack ? 0 : qt * 32) + off, pos_hi = (p.pack ? p.Tq - 1 : min(qt * 32 + 31, p.Tq - 1)) + off;
  const T* kb = reinterpret_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h;
  const T* vb = reinterpret_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h;
  const uint8_t* mask = p.key_mask ? p.key_mask + b * p.mask_b : nullptr;
  Stationary<T, DP, false> q;
  q.load(reinterpret_cast<const T*>(p.q) + b * p.q_b + h * p.q_h + min(qi, p.Tq - 1) * p.q_t, half, p.D, p.vec, true);
  const int lut_len = 2 * p.max_distance + 1;
  if constexpr (BIAS) {
    if (p.pack)
      for (int g = 0; g < p.group; ++g) fill_lut(p, hh * p.group + g, lut + g * lut_len, tid, 256);
    else
      fill_lut(p, h, lut, tid, 256);
  }
  const int end = key_end(p, b, pos_hi, word, tid, 256);
  const int all = (end + 31) / 32, per = (all + p.splits - 1) / p.splits, t1 = min(all, (split + 1) * per);
  if constexpr (BIAS) __syncthreads();
  const float* my_lut = lut + (p.pack ? min(lh, p.group - 1) * lut_len : 0);

  f32x16 acc[DT] = {};
  Running run;
  Raw<T> k[NC2], v[VP][NV];
  uint64_t keys = 0;  // of the requested tile: bit r = key r may be used
  auto load_k = [&](int t) {
    const int row = t * 32 + col, rc = min(row, end - 1);
    keys = __ballot(row < end && !(mask && mask[rc]));
    const T* kr = kb + rc * p.k_t;
#pragma unroll
    for (int c = 0; c < NC2; ++c) k[c] = load_chunk<T>(kr, 2 * c + half, p.D, p.vec);
  };
  auto load_v = [&](int t, int part) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int id = i * 64 + lane, vr = t * 32 + id / NCV;
      v[part][i] = load_chunk<T>(vb + min(vr, end - 1) * p.v_t, part * NCV + id % NCV, p.D, p.vec);
    }
  };
  int t = split * per + wave;
  if (t < t1) {
    load_k(t);
    if (AHEAD)
#pragma unroll
      for (int part = 0; part < VP; ++part) load_v(t, part);
  }
  for (; t < t1; t += 4) {
    const int key0 = t * 32;
    const uint32_t use = (uint32_t)keys;
    f32x16 raw = {};
    if (use != ~0u && !((use >> col) & 1)) {
#pragma unroll
      for (int c = 0; c < NC2; ++c) k[c].x = {};
    }
#pragma unroll
    for (int c = 0; c < NC2; ++c) raw = mma(operand(k[c]), q.get(c), raw);
    float s[1][16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = raw[i];
    if (t + 4 < t1) load_k(t + 4);
    finish_scores<BIAS>(p, s[0], key0, pos, pos_lo, pos_hi, use, my_lut, half);
    run.step(s, acc);
    const Weights<T> w(s[0]);
#pragma unroll
    for (int part = 0; part < VP; ++part) {
      if (!AHEAD) load_v(t, part);
      // LDS operations of a wave stay in order: the last reads of the private tile come before these writes
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int vr = (i * 64 + lane) / NCV;
        if (use != ~0u && !((use >> vr) & 1)) v[part][i].x = {};
        TL::put(vt, vr, (i * 64 + lane) % NCV, operand(v[part][i]));
      }
      if (AHEAD && t + 4 < t1) load_v(t + 4, part);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      f32x16(&mine)[DV / 32] = *reinterpret_cast<f32x16(*)[DV / 32]>(&acc[part * (DV / 32)]);
      column_product<T, TL>(vt, 0, 0, w, mine, lane);
    }
  }
  // join the four waves: a common maximum per column, then sums over the waves in their order
  const float l = both_sum(run.l);
  if (half == 0) {
    ml[(wave * 2) * 32 + col] = run.m;
    ml[(wave * 2 + 1) * 32 + col] = l;
  }
  __syncthreads();
  float m = ml[col];
#pragma unroll
  for (int w = 1; w < 4; ++w) m = fmaxf(m, ml[(w * 2) * 32 + col]);
  const float a = exp2f(run.m - m);
  constexpr int LD = DP + 4;
  float* mine = reinterpret_cast<float*>(vt);  // [32][LD], the wave's own tile is done with
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(mine + col * LD + dt * 32 + 8 * g + 4 * half) =
          f32x4{acc[dt][4 * g] * a, acc[dt][4 * g + 1] * a, acc[dt][4 * g + 2] * a, acc[dt][4 * g + 3] * a};
  __syncthreads();
  // eight threads a column
  const int c2 = tid >> 3;
  float m2 = ml[c2], l2 = 0.f;
#pragma unroll
  for (int w = 1; w < 4; ++w) m2 = fmaxf(m2, ml[(w * 2) * 32 + c2]);
#pragma unroll
  for (int w = 0; w < 4; ++w) l2 += ml[(w * 2 + 1) * 32 + c2] * exp2f(ml[(w * 2) * 32 + c2] - m2);
  const int lh2 = p.pack ? c2 / p.Tq : 0, h2 = p.pack ? hh * p.group + lh2 : hh, qi2 = p.pack ? c2 - lh2 * p.Tq : qt * 32 + c2;
  if (p.pack ? lh2 >= p.group : qi2 >= p.Tq) return;
  const int64_t row = ((int64_t)b * p.H + h2) * p.Tq + qi2;
  auto sum = [&](int d) {
    f32x4 x = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) x += *reinterpret_cast<const f32x4*>(smem + w * split_wave_bytes<T, DP>() + (c2 * LD + d) * 4);
    return x;
  };
  if (p.splits == 1) {
    const float inv = l2 > 0.f ? 1.f / l2 : (l2 == 0.f ? 0.f : l2);
    T* orow = reinterpret_cast<T*>(p.out) + b * p.o_b + h2 * p.o_h + qi2 * p.o_t;
    for (int d = (tid & 7) * 4; d < DP; d += 32) {
      const f32x4 x = sum(d);
      store4<T>(orow, d, p.D, p.vec, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    }
    if ((tid & 7) == 0 && p.lse) p.lse[row] = l2 == 0.f ? -INFINITY : (m2 + log2f(l2)) * kLn2;
  } else {
    float* part = p.part + (row * p.splits + split) * (DP + 4);
    for (int d = (tid & 7) * 4; d < DP; d += 32) *reinterpret_cast<f32x4*>(part + 4 + d) = sum(d);
    if ((tid & 7) == 0) {
      part[0] = m2;
      part[1] = l2;
    }
  }
}

// Joins the splits of a query: one wave per query, splits in their order.
template <class T, int DP>
__global__ __launch_bounds__(256) void attention_join_kernel(Params p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)p.B * p.H * p.Tq) return;
  const float* part = p.part + row * p.splits * (DP + 4);
  float m = -3e38f, l = 0.f;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, part[s * (DP + 4)]);
  constexpr int E = DP / 64;
  float x[E] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float* ps = part + s * (DP + 4);
    const float a = exp2f(ps[0] - m);
    l += ps[1] * a;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] += ps[4 + e * 64 + lane] * a;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int qi = row % p.Tq, h = (row / p.Tq) % p.H, b = row / p.Tq / p.H;
  T* orow = reinterpret_cast<T*>(p.out) + b * p.o_b + h * p.o_h + qi * p.o_t;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e * 64 + lane < p.D) orow[e * 64 + lane] = (T)(x[e] * inv);
  if (lane == 0 && p.lse) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// ------------------------------------------------------------------ host

constexpr int kComputeUnits = 256;

static int padded_dim(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
static int lut_floats(const Params& p) { return p.table ? 2 * p.max_distance + 1 : 0; }

// How a call runs.  The 128-query kernel shares each key tile among four waves and is the faster one as soon as its workgroups
// fill the compute units; below that the split kernel has four times the workgroups and can divide the keys too.
static void plan(Params* p) {
  const int64_t wide = (int64_t)p->B * p->H * ((p->Tq + 127) / 128);
  p->splits = 0;
  p->pack = 0;
  if (wide >= kComputeUnits && p->Tq > 32) return;
  p->pack = (int64_t)p->group * p->Tq <= 32 && (size_t)p->group * lut_floats(*p) * 4 <= 16 * 1024;
  const int64_t base = p->pack ? (int64_t)p->B * p->Hkv : (int64_t)p->B * p->H * ((p->Tq + 31) / 32);
  const int64_t rounds = (p->Tk + 127) / 128;  // a wave's tiles if the keys are not split
  int64_t s = (2 * kComputeUnits + base - 1) / base;
  if (s > (rounds + 1) / 2) s = (rounds + 1) / 2;
  p->splits = (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

static size_t split_workspace(const Params& p) {
  return p.splits > 1 ? (size_t)p.B * p.H * p.Tq * p.splits * (padded_dim(p.D) + 4) * sizeof(float) : 0;
}

template <class T, int DP, bool BIAS>
static int launch_forward(const Params& p, hipStream_t st) {
  static std::atomic<uint64_t> wide_done{0}, split_done{0};
  const size_t lut = BIAS ? lut_floats(p) * sizeof(float) : 0;
  if (p.splits == 0) {
    return launch(&attention_forward_kernel<T, DP, BIAS>, &wide_done, (int64_t)p.B * p.H * ((p.Tq + 127) / 128),
                  2 * forward_buffers<T, DP>() * Tile<T, DP, key_tile<T>()>::BYTES + 16 + lut, p, st);
  }
  const int64_t n = (p.pack ? (int64_t)p.B * p.Hkv : (int64_t)p.B * p.H * ((p.Tq + 31) / 32)) * p.splits;
  if (launch(&attention_split_kernel<T, DP, BIAS>, &split_done, n,
             4 * split_wave_bytes<T, DP>() + 4 * 2 * 32 * 4 + 16 + lut * (p.pack ? p.group : 1), p, st))
    return 1;
  if (p.splits > 1) {
    const int64_t rows = (int64_t)p.B * p.H * p.Tq;
    hipLaunchKernelGGL((attention_join_kernel<T, DP>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
    WRNN_LAUNCH_CHECK();
  }
  return 0;
}

template <class T, int DP>
static int launch_bias(const Params& p, hipStream_t st) {
  return p.table ? launch_forward<T, DP, true>(p, st) : launch_forward<T, DP, false>(p, st);
}

template <class T>
static int launch_dim(const Params& p, hipStream_t st) {
  switch (padded_dim(p.D)) {
    case 64: return launch_bias<T, 64>(p, st);
    case 128: return launch_bias<T, 128>(p, st);
    default: return launch_bias<T, 256>(p, st);
  }
}

}  // namespace attn

int attention_params(const wrnn_attention_desc* d, attn::Params* p, const char* who) {
  using namespace attn;
  WRNN_REQUIRE(d, "%s: null description", who);
  WRNN_REQUIRE(d->dtype == WRNN_FLOAT32 || d->dtype == WRNN_BFLOAT16, "%s: dtype %d is neither float32 nor bfloat16", who, d->dtype);
  WRNN_REQUIRE(d->batch >= 0 && d->heads >= 0 && d->kv_heads >= 0 && d->q_len >= 0 && d->k_len >= 0, "%s: negative size", who);
  WRNN_REQUIRE(d->head_dim >= 1 && d->head_dim <= 256, "%s: head dimension %d is outside 1 .. 256", who, d->head_dim);
  WRNN_REQUIRE(d->q_len <= (1 << 28) && d->k_len <= (1 << 28), "%s: sequences are at most 2^28 long", who);
  WRNN_REQUIRE(d->heads == 0 || (d->kv_heads > 0 && d->heads % d->kv_heads == 0), "%s: %d heads do not share %d key heads evenly", who,
               d->heads, d->kv_heads);
  const int64_t tiles = (int64_t)d->batch * d->heads * ((d->q_len > d->k_len ? d->q_len : d->k_len) / 32 + 1);
  WRNN_REQUIRE(tiles < (1LL << 22), "%s: batch x heads x length is too large for one launch", who);
  const bool some = d->batch && d->heads && d->q_len;
  WRNN_REQUIRE(!some || (d->q && (d->k_len == 0 || (d->k && d->v))), "%s: null pointer", who);
  *p = Params{};
  // a stride over a dimension of one is never taken: whatever it says, it does not decide about alignment
  auto st = [](int n, int64_t s) { return n > 1 ? s : 0; };
  p->q = d->q, p->k = d->k, p->v = d->v;
  p->q_b = st(d->batch, d->q_stride[0]), p->q_h = st(d->heads, d->q_stride[1]), p->q_t = st(d->q_len, d->q_stride[2]);
  p->k_b = st(d->batch, d->k_stride[0]), p->k_h = st(d->kv_heads, d->k_stride[1]), p->k_t = st(d->k_len, d->k_stride[2]);
  p->v_b = st(d->batch, d->v_stride[0]), p->v_h = st(d->kv_heads, d->v_stride[1]), p->v_t = st(d->k_len, d->v_stride[2]);
  // a lane's rows inside a tile are found with 32-bit offsets
  for (int64_t s : {p->q_t, p->k_t, p->v_t})
    WRNN_REQUIRE(s > -kMaxRowStride && s < kMaxRowStride, "%s: position strides are below 2^26 elements", who);
  p->B = d->batch, p->H = d->heads, p->Hkv = d->kv_heads, p->group = d->heads ? d->heads / d->kv_heads : 1;
  p->Tq = d->q_len, p->Tk = d->k_len, p->D = d->head_dim;
  p->causal = d->causal != 0;
  p->scale = d->scale, p->scale2 = d->scale * kLog2e;
  p->key_mask = d->key_mask, p->mask_b = d->key_mask_stride, p->key_lens = d->key_lens, p->q_start = d->q_start;
  const int es = d->dtype == WRNN_FLOAT32 ? 4 : 2;
  p->vec = d->head_dim % (16 / es) == 0 && rows_on_16(p->q, p->q_b, p->q_h, p->q_t, es) && rows_on_16(p->k, p->k_b, p->k_h, p->k_t, es) &&
           rows_on_16(p->v, p->v_b, p->v_h, p->v_t, es);
  if (d->bias_table) {
    if (bias_params(p, d->num_buckets, d->max_distance, d->bidirectional, d->bucket_edges, who)) return 1;
    p->table = d->bias_table;
  }
  return 0;
}

}  // namespace wrnn

using namespace wrnn;

extern "C" size_t wrnn_attention_workspace_bytes(const wrnn_attention_desc* desc) {
  attn::Params p;
  if (attention_params(desc, &p, "wrnn_attention_workspace_bytes") || !p.B || !p.H || !p.Tq) return 0;
  attn::plan(&p);
  return attn::split_workspace(p);
}

extern "C" int wrnn_attention_forward(const wrnn_attention_desc* desc, void* out, const int64_t out_stride[3], float* lse, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  attn::Params p;
  if (attention_params(desc, &p, "wrnn_attention_forward")) return 1;
  if (!p.B || !p.H || !p.Tq) return 0;
  WRNN_REQUIRE(out && out_stride, "wrnn_attention_forward: null pointer");
  attn::plan(&p);
  const size_t need = attn::split_workspace(p);
  WRNN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "wrnn_attention_forward: workspace of %zu bytes, %zu are needed",
               workspace_bytes, need);
  p.out = out, p.o_b = out_stride[0], p.o_h = out_stride[1], p.o_t = out_stride[2], p.lse = lse;
  p.part = static_cast<float*>(workspace);
  const int es = desc->dtype == WRNN_FLOAT32 ? 4 : 2;
  p.vec = p.vec && attn::rows_on_16(out, p.o_b, p.o_h, p.o_t, es);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return desc->dtype == WRNN_FLOAT32 ? attn::launch_dim<float>(p, st) : attn::launch_dim<__bf16>(p, st);
}
