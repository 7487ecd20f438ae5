// The learned relative position bias as a dense tensor, and its table's gradient.
//   out[h, i, j] = table[bucket(j - (i + start)), h]          bound by the writes of H * Tq * Tk values: 16 x 2048 x 2048 in float32 in 41 us,
//                                                              6.5 TB/s (filling as much memory 6.9)
//   dtable[n, h] = sum over the pairs of bucket n of dout      bound by the reads of them: the same 75 us, 3.6 TB/s (a plain sum 4.0)
// A bucket depends on the distance alone and is constant from max_distance on, so both work on one value per distance in
// [-max_distance, max_distance] (LDS) and never look at a bucket inside the loops.
#include "attention_tile.h"

namespace wrnn {
namespace attn {

// the arguments beyond the bucket rule (Params)
struct DenseBias {
  const void* in;  // table, or dout
  void* out;
  float* part;
  int start, rows;  // rows of a workgroup
};

// One wave per row: 16-byte stores from the row's first aligned element on, single ones before and behind.
template <class T>
__global__ __launch_bounds__(256) void relative_bias_kernel(Params p, DenseBias a) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V)));
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* lut = reinterpret_cast<T*>(smem);
  const int tid = threadIdx.x, lane = tid & 63, md = p.max_distance;
  const int chunks = (p.Tq + a.rows - 1) / a.rows, h = blockIdx.x / chunks, i0 = (blockIdx.x - h * chunks) * a.rows;
  const T* table = reinterpret_cast<const T*>(a.in);
  for (int i = tid; i <= 2 * md; i += 256) lut[i] = table[(int64_t)bucket_of(p, i - md) * p.H + h];
  __syncthreads();
  for (int i = i0 + (tid >> 6); i < min(i0 + a.rows, p.Tq); i += 4) {
    T* row = reinterpret_cast<T*>(a.out) + ((int64_t)h * p.Tq + i) * p.Tk;
    const int pos = i + a.start;
    auto at = [&](int j) { return lut[min(max(j - pos, -md), md) + md]; };
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T), p.Tk);
    const int full = (p.Tk - head) / V;
    for (int c = lane; c < full; c += 64) {
      const int j = head + c * V;
      vec x;
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = at(j + e);
      *reinterpret_cast<vec*>(row + j) = x;
    }
    if (lane < head) row[lane] = at(lane);
    const int tail = head + full * V + lane;
    if (lane < V && tail < p.Tk) row[tail] = at(tail);
  }
}

// A workgroup's rows -> one partial sum per bucket.  Near the diagonal a thread owns a distance and walks the rows; what lies further out a wave
// reads row by row, four rows at a time to have enough loads in flight, 16 bytes a load from each row's first aligned element on (the
// vectors that lie wholly near the diagonal are left to the walk).  Nothing is read twice: loads that leave the caches alone are the faster
// (16 x 2048 x 2048 and 2047 x 2047 with the forward pass 140 and 150 -> 122 and 119 us).
template <class T>
__global__ __launch_bounds__(256) void relative_bias_grad_kernel(Params p, DenseBias a) {
  constexpr int V = 16 / sizeof(T), R = 4;
  typedef T vec __attribute__((ext_vector_type(V)));
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* sums = reinterpret_cast<float*>(smem);  // [2 * max_distance + 1]
  float* ends = sums + 2 * p.max_distance + 1;   // [4][2]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), md = p.max_distance;
  const int chunks = (p.Tq + a.rows - 1) / a.rows, h = blockIdx.x / chunks, i0 = (blockIdx.x - h * chunks) * a.rows,
            i1 = min(i0 + a.rows, p.Tq);
  const T* base = reinterpret_cast<const T*>(a.in) + (int64_t)h * p.Tq * p.Tk;
  float below[R] = {}, above[R] = {};
  for (int i = i0 + wave * R; i < i1; i += 4 * R) {
    const T* row[R];
    int head[R], full[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      row[r] = base + (int64_t)min(i + r, i1 - 1) * p.Tk;
      head[r] = min((int)((16 - (reinterpret_cast<uintptr_t>(row[r]) & 15)) & 15) / (int)sizeof(T), p.Tk);
      full[r] = i + r < i1 ? (p.Tk - head[r]) / V : 0;
    }
    auto put = [&](int r, int rel, float x) {
      below[r] += rel <= -md ? x : 0.f;
      above[r] += rel >= md ? x : 0.f;
    };
    const int most = (p.Tk + V - 1) / V;
#pragma unroll 2
    for (int c = lane; c < most; c += 64) {
      vec v[R];
      int rel[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = head[r] + c * V;
        rel[r] = j - (i + r + a.start);
        v[r] = vec(T(0));
        if (c < full[r] && !(rel[r] > -md && rel[r] + V - 1 < md)) v[r] = __builtin_nontemporal_load(reinterpret_cast<const vec*>(row[r] + j));
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) put(r, rel[r] + e, (float)v[r][e]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (i + r >= i1) break;
      const int pos = i + r + a.start, tail = head[r] + full[r] * V + lane;
      if (lane < head[r]) put(r, lane - pos, (float)row[r][lane]);
      if (lane < V && tail < p.Tk) put(r, tail - pos, (float)row[r][tail]);
    }
  }
  float lo = below[0], hi = above[0];
#pragma unroll
  for (int r = 1; r < R; ++r) lo += below[r], hi += above[r];
  for (int r = 1 - md + tid; r < md; r += 256) {
    float x = 0.f;
#pragma unroll 16
    for (int i = i0; i < i1; ++i) {
      const int j = i + a.start + r;
      if (j >= 0 && j < p.Tk) x += (float)base[(int64_t)i * p.Tk + j];
    }
    sums[r + md] = x;
  }
  for (int m = 1; m < 64; m <<= 1) {
    lo += __shfl_xor(lo, m);
    hi += __shfl_xor(hi, m);
  }
  if (lane == 0) {
    ends[2 * wave] = lo;
    ends[2 * wave + 1] = hi;
  }
  __syncthreads();
  if (tid < 2) sums[tid * 2 * md] = ends[tid] + ends[2 + tid] + ends[4 + tid] + ends[6 + tid];
  __syncthreads();
  if (tid < p.buckets) a.part[((int64_t)(blockIdx.x - h * chunks) * p.H + h) * p.buckets + tid] = bucket_sum(p, sums, tid);
}

// One wave per (bucket, head): lanes take the partial sums in turn, then a fixed tree.
template <class T>
__global__ __launch_bounds__(64) void table_sum_kernel(const float* part, int rows, int H, int buckets, T* dtable) {
  const int n = blockIdx.x % buckets, h = blockIdx.x / buckets;
  double x = 0.;
  for (int r = threadIdx.x; r < rows; r += 64) x += part[((int64_t)r * H + h) * buckets + n];
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
  if (threadIdx.x == 0) dtable[(int64_t)n * H + h] = (T)(float)x;
}

// ------------------------------------------------------------------ host

template <class T>
int launch_table_sum(const float* part, int rows, int H, int buckets, T* dtable, hipStream_t st) {
  hipLaunchKernelGGL((table_sum_kernel<T>), dim3(buckets * H), dim3(64), 0, st, part, rows, H, buckets, dtable);
  WRNN_LAUNCH_CHECK();
  return 0;
}
template int launch_table_sum<float>(const float*, int, int, int, float*, hipStream_t);

int bias_params(Params* p, int num_buckets, int max_distance, int bidirectional, const int32_t* edges, const char* who) {
  const int side = bidirectional ? num_buckets / 2 : num_buckets, n = side - side / 2 - 1;
  WRNN_REQUIRE(num_buckets >= 2 && num_buckets <= 256 && (!bidirectional || (num_buckets % 2 == 0 && side >= 2)),
               "%s: %d buckets: 2 .. 256 are served, 4 .. 256 and an even number with two sides", who, num_buckets);
  WRNN_REQUIRE((int64_t)p->H * num_buckets < (1LL << 26), "%s: heads x buckets is too large for one launch", who);
  WRNN_REQUIRE(max_distance > side / 2 && max_distance <= kMaxDistance, "%s: max_distance %d is outside %d .. %d", who, max_distance,
               side / 2 + 1, kMaxDistance);
  WRNN_REQUIRE(n <= kMaxEdges && (n == 0 || edges), "%s: null bucket edges", who);
  for (int i = 0; i < n; ++i) {
    WRNN_REQUIRE(edges[i] >= (i ? edges[i - 1] : side / 2) && edges[i] <= max_distance,
                 "%s: bucket edges have to ascend from %d to max_distance", who, side / 2);
    p->edges[i] = edges[i];
  }
  p->buckets = num_buckets, p->max_distance = max_distance, p->two_sided = bidirectional != 0;
  p->exact_side = side / 2, p->side = side, p->n_edges = n;
  return 0;
}

// Rows of a workgroup: enough that its table of distances is small beside them, few enough that the compute units are filled.
static int bias_rows(int heads, int q_len, int k_len) {
  const int64_t want = (int64_t)heads * q_len / 1024;
  const int64_t most = k_len >= 512 ? 32 : 64;
  return (int)(want < 4 ? 4 : want > most ? most : (want + 3) / 4 * 4);
}

static int dense_params(Params* p, int dtype, int heads, int q_len, int k_len, int start, int num_buckets, int max_distance, int bidirectional,
                        const int32_t* edges, const char* who) {
  *p = Params{};
  WRNN_REQUIRE(dtype == WRNN_FLOAT32 || dtype == WRNN_BFLOAT16, "%s: dtype %d is neither float32 nor bfloat16", who, dtype);
  WRNN_REQUIRE(heads >= 0 && q_len >= 0 && k_len >= 0, "%s: negative size", who);
  WRNN_REQUIRE(q_len <= (1 << 28) && k_len <= (1 << 28) && start >= -(1 << 29) && start <= (1 << 29), "%s: lengths are at most 2^28, start 2^29",
               who);
  const int64_t rows = bias_rows(heads, q_len, k_len);
  WRNN_REQUIRE(heads * ((q_len + rows - 1) / rows) * 256 < (1LL << 32), "%s: heads x q_len is too large for one launch", who);
  p->H = heads, p->Tq = q_len, p->Tk = k_len;
  return bias_params(p, num_buckets, max_distance, bidirectional, edges, who);
}

}  // namespace attn
}  // namespace wrnn

using namespace wrnn;

extern "C" int wrnn_relative_bias_forward(const void* table, int dtype, int heads, int q_len, int k_len, int start, int num_buckets,
                                          int max_distance, int bidirectional, const int32_t* bucket_edges, void* out, void* stream) {
  attn::Params p;
  if (attn::dense_params(&p, dtype, heads, q_len, k_len, start, num_buckets, max_distance, bidirectional, bucket_edges, "wrnn_relative_bias_forward"))
    return 1;
  if (!heads || !q_len || !k_len) return 0;
  WRNN_REQUIRE(table && out, "wrnn_relative_bias_forward: null pointer");
  attn::DenseBias a{table, out, nullptr, start, attn::bias_rows(heads, q_len, k_len)};
  const unsigned grid = (unsigned)(heads * ((q_len + a.rows - 1) / a.rows));
  const size_t lds = (size_t)(2 * max_distance + 1) * (dtype == WRNN_FLOAT32 ? 4 : 2);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == WRNN_FLOAT32)
    hipLaunchKernelGGL((attn::relative_bias_kernel<float>), dim3(grid), dim3(256), lds, st, p, a);
  else
    hipLaunchKernelGGL((attn::relative_bias_kernel<__bf16>), dim3(grid), dim3(256), lds, st, p, a);
  WRNN_LAUNCH_CHECK();
  return 0;
}

extern "C" size_t wrnn_relative_bias_workspace_bytes(int heads, int q_len, int k_len, int num_buckets, int max_distance) {
  (void)max_distance;
  if (heads <= 0 || q_len <= 0 || k_len <= 0 || num_buckets <= 0) return 0;
  const int rows = attn::bias_rows(heads, q_len, k_len);
  return (size_t)((q_len + rows - 1) / rows) * heads * num_buckets * sizeof(float);
}

extern "C" int wrnn_relative_bias_backward(const void* dout, int dtype, int heads, int q_len, int k_len, int start, int num_buckets,
                                           int max_distance, int bidirectional, const int32_t* bucket_edges, void* dtable, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  attn::Params p;
  if (attn::dense_params(&p, dtype, heads, q_len, k_len, start, num_buckets, max_distance, bidirectional, bucket_edges, "wrnn_relative_bias_backward"))
    return 1;
  if (!heads) return 0;
  WRNN_REQUIRE(dtable && q_len && k_len, "wrnn_relative_bias_backward: null gradient, or no pairs (the gradient is zero and left to the caller)");
  const size_t need = wrnn_relative_bias_workspace_bytes(heads, q_len, k_len, num_buckets, max_distance);
  WRNN_REQUIRE(dout && workspace && workspace_bytes >= need, "wrnn_relative_bias_backward: workspace of %zu bytes, %zu are needed", workspace_bytes,
               need);
  attn::DenseBias a{dout, nullptr, static_cast<float*>(workspace), start, attn::bias_rows(heads, q_len, k_len)};
  const int chunks = (q_len + a.rows - 1) / a.rows;
  const size_t lds = (size_t)(2 * max_distance + 1 + 8) * 4;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == WRNN_FLOAT32)
    hipLaunchKernelGGL((attn::relative_bias_grad_kernel<float>), dim3((unsigned)(heads * chunks)), dim3(256), lds, st, p, a);
  else
    hipLaunchKernelGGL((attn::relative_bias_grad_kernel<__bf16>), dim3((unsigned)(heads * chunks)), dim3(256), lds, st, p, a);
  WRNN_LAUNCH_CHECK();
  return dtype == WRNN_FLOAT32 ? attn::launch_table_sum<float>(a.part, chunks, heads, num_buckets, static_cast<float*>(dtable), st)
                               : attn::launch_table_sum<__bf16>(a.part, chunks, heads, num_buckets, static_cast<__bf16*>(dtable), st);
}
