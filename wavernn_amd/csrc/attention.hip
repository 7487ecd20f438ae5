// Entry points of the self-attention (kernels: attention_forward.h, attention_backward.h; several sources for the build's sake).
#include <cmath>

#include "attention_tile.h"

namespace wrnn {
namespace attn {

template <class T, int DP>
int forward(const Params& p, hipStream_t st);
template <class T, int DP>
int backward(const Params& p, float* dtable, hipStream_t st);

template <class T>
static int forward(const Params& p, hipStream_t st) {
  return p.D <= 64 ? forward<T, 64>(p, st) : p.D <= 128 ? forward<T, 128>(p, st) : forward<T, 256>(p, st);
}
template <class T>
static int backward(const Params& p, float* dtable, hipStream_t st) {
  return p.D <= 64 ? backward<T, 64>(p, dtable, st) : p.D <= 128 ? backward<T, 128>(p, dtable, st) : backward<T, 256>(p, dtable, st);
}

constexpr int kComputeUnits = 256;

static int padded_dim(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
static int lut_floats(const Params& p) { return p.table ? 2 * p.max_distance + 1 : 0; }

// Workgroups that share one block of stationary rows, each with part of the `tiles` of the other side: as many as fill the compute units,
// none with fewer than `least` tiles (1 x 2 heads, 128 x 128 x 128 in bfloat16: 13.5 us undivided, 17.7 with shares of two tiles, for the joining
// launch).  Where the blocks alone fill the compute units one and a bit times, dividing them evens the last round out but
// costs more than that gives: 32 x 2 heads, 640 x 640 x 128 in float32 102 us, 121 with two shares, 119 with three.  A compute unit counts as one
// place, also for the kernels of which it holds two.
static int shares(int64_t blocks, int64_t tiles, int least) {
  const int64_t want = kComputeUnits / (blocks > 0 ? blocks : 1), most = tiles / least;
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

// How a call runs.  The wide shape shares each key tile among four waves; the narrow one is for few queries, which would leave three of
// them idle (one query, 8 x 16 heads, 4096 keys of 128 columns in bfloat16: 49 us narrow, 56 wide; 20 queries at 64 columns 27 and 39; one in
// float32, 2048 keys 42 and 58).  Heads that share k and v become columns of one tile where all their queries fit it and their bias tables leave
// room: the cache is read once (one query, 8 x 16 heads on 4, 8191 keys: 31 us, head by head 49).
static void plan(Params* p) {
  p->pack = p->group > 1 && (int64_t)p->group * p->Tq <= 32 && (size_t)p->group * lut_floats(*p) * 4 <= 16 * 1024;
  p->narrow = p->pack || p->Tq <= 32;
  if (p->narrow) {
    const int64_t blocks = p->pack ? (int64_t)p->B * p->Hkv : (int64_t)p->B * p->H;
    p->splits = shares((blocks + 1) / 2, (p->Tk + 127) / 128, 2);
  } else {
    p->splits = shares((int64_t)p->B * p->H * ((p->Tq + 127) / 128), (p->Tk + 31) / 32, 4);
  }
}
static size_t split_workspace(const Params& p) {
  return p.splits > 1 ? (size_t)p.B * p.H * p.Tq * p.splits * (padded_dim(p.D) + 4) * sizeof(float) : 0;
}

// blocks of a workgroup's rows: two waves share a row past 128 columns (BackwardShape)
static int row_blocks(const Params& p, int rows) { return p.D > 128 ? (rows + 63) / 64 : (rows + 127) / 128; }
static void plan_backward(Params* p, int dtype) {
  // (bfloat16 with few keys: the joining launch costs what shares would save)
  p->dq_splits = dtype == WRNN_BFLOAT16 && p->Tk <= 512 ? 1 : shares((int64_t)p->B * p->H * row_blocks(*p, p->Tq), (p->Tk + 31) / 32, 4);
  // (causality: the first keys' blocks are the longest by far; half as long they leave the others time to fill up)
  const int64_t blocks = (int64_t)p->B * p->Hkv * row_blocks(*p, p->Tk);
  p->dkv_splits = shares(p->causal ? (blocks + 1) / 2 : blocks, (int64_t)((p->Tq + 31) / 32) * p->group, 4);
}
static size_t aligned(size_t x) { return (x + 255) & ~size_t(255); }
// the backward workspace: the rows' statistics, delta, the table's partial sums, the shares
static size_t stats_bytes(const Params& p) { return aligned((size_t)2 * p.B * p.H * p.Tq * sizeof(float)); }
static size_t delta_bytes(const Params& p, int dtype) {
  return aligned((size_t)(p.table || dtype == WRNN_BFLOAT16 ? p.dq_splits : 1) * p.B * p.H * p.Tq * sizeof(float));
}
static size_t table_bytes(const Params& p) {
  return p.table ? aligned((size_t)p.B * row_blocks(p, p.Tk) * p.dkv_splits * p.H * p.buckets * sizeof(float)) : 0;
}
static size_t dq_bytes(const Params& p) { return p.dq_splits > 1 ? aligned((size_t)p.dq_splits * p.B * p.H * p.Tq * p.D * sizeof(float)) : 0; }
static size_t dkv_bytes(const Params& p) { return p.dkv_splits > 1 ? (size_t)p.dkv_splits * 2 * p.B * p.Hkv * p.Tk * p.D * sizeof(float) : 0; }

// a stride over a dimension of one is never taken: whatever it says, it does not decide about alignment
static int64_t stride_of(int n, int64_t s) { return n > 1 ? s : 0; }

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
  p->q = d->q, p->k = d->k, p->v = d->v;
  p->q_b = stride_of(d->batch, d->q_stride[0]), p->q_h = stride_of(d->heads, d->q_stride[1]), p->q_t = stride_of(d->q_len, d->q_stride[2]);
  p->k_b = stride_of(d->batch, d->k_stride[0]), p->k_h = stride_of(d->kv_heads, d->k_stride[1]), p->k_t = stride_of(d->k_len, d->k_stride[2]);
  p->v_b = stride_of(d->batch, d->v_stride[0]), p->v_h = stride_of(d->kv_heads, d->v_stride[1]), p->v_t = stride_of(d->k_len, d->v_stride[2]);
  // a lane's rows inside a tile are found with 32-bit offsets
  for (int64_t s : {p->q_t, p->k_t, p->v_t})
    WRNN_REQUIRE(s >= 0 && s < kMaxRowStride, "%s: position strides are in 0 .. 2^22 - 1 elements", who);
  p->B = d->batch, p->H = d->heads, p->Hkv = d->kv_heads, p->group = d->heads ? d->heads / d->kv_heads : 1;
  p->Tq = d->q_len, p->Tk = d->k_len, p->D = d->head_dim;
  p->causal = d->causal != 0;
  // the kernels take the scale as positive (the highest product is the highest score) and not zero, which a left out pair's -inf would not survive
  p->scale = d->scale, p->flip = d->scale < 0.f ? 0x80000000u : 0u;
  p->scale2 = d->scale == 0.f ? 1.17549435e-38f : std::fabs(d->scale) * kLog2e;
  p->key_mask = d->key_mask, p->mask_b = d->key_mask_stride, p->key_lens = d->key_lens, p->q_start = d->q_start;
  const int es = d->dtype == WRNN_FLOAT32 ? 4 : 2;
  WRNN_REQUIRE(d->head_dim % 4 == 0 && d->head_dim * es >= 16 && rows_on_four(p->q, p->q_b, p->q_h, p->q_t, es) &&
                   rows_on_four(p->k, p->k_b, p->k_h, p->k_t, es) && rows_on_four(p->v, p->v_b, p->v_h, p->v_t, es),
               "%s: rows have to hold whole fours of elements, 16 bytes at least, and start on the bytes of four", who);
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
  return wrnn_attention_forward_stats(desc, out, out_stride, lse, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int wrnn_attention_forward_stats(const wrnn_attention_desc* desc, void* out, const int64_t out_stride[3], float* lse, float* stats,
                                            void* workspace, size_t workspace_bytes, void* stream) {
  attn::Params p;
  if (attention_params(desc, &p, "wrnn_attention_forward")) return 1;
  if (!p.B || !p.H || !p.Tq) return 0;
  WRNN_REQUIRE(out && out_stride, "wrnn_attention_forward: null pointer");
  attn::plan(&p);
  const size_t need = attn::split_workspace(p);
  WRNN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && !((uintptr_t)workspace & 15)),
               "wrnn_attention_forward: workspace of %zu bytes, %zu are needed, on 16 bytes", workspace_bytes, need);
  p.out = out, p.lse = lse, p.stats = stats;
  p.o_b = attn::stride_of(p.B, out_stride[0]), p.o_h = attn::stride_of(p.H, out_stride[1]), p.o_t = attn::stride_of(p.Tq, out_stride[2]);
  p.part = static_cast<float*>(workspace);
  WRNN_REQUIRE(attn::rows_on_four(out, p.o_b, p.o_h, p.o_t, desc->dtype == WRNN_FLOAT32 ? 4 : 2), "wrnn_attention_forward: rows of out have to start on the bytes of four elements");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return desc->dtype == WRNN_FLOAT32 ? attn::forward<float>(p, st) : attn::forward<__bf16>(p, st);
}

extern "C" size_t wrnn_attention_backward_workspace_bytes(const wrnn_attention_desc* desc) {
  attn::Params p;
  if (attention_params(desc, &p, "wrnn_attention_backward_workspace_bytes") || !p.B || !p.H || !p.Tq) return 0;
  attn::plan(&p);
  attn::plan_backward(&p, desc->dtype);
  const size_t rest = attn::delta_bytes(p, desc->dtype) + attn::table_bytes(p) + attn::dq_bytes(p) + attn::dkv_bytes(p), forward = attn::split_workspace(p);
  return attn::stats_bytes(p) + (rest > forward ? rest : forward);
}

extern "C" int wrnn_attention_backward(const wrnn_attention_desc* desc, const wrnn_attention_grads* g, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  return wrnn_attention_backward_stats(desc, g, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int wrnn_attention_backward_stats(const wrnn_attention_desc* desc, const wrnn_attention_grads* g, const float* stats, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  attn::Params p;
  if (attention_params(desc, &p, "wrnn_attention_backward")) return 1;
  WRNN_REQUIRE(g, "wrnn_attention_backward: null gradients");
  if (!p.B || !p.H || !p.Tq) {
    WRNN_REQUIRE(!p.B || !p.H || !p.Tk, "wrnn_attention_backward: no queries; dk, dv and the table's gradient are zero and left to the caller");
    return 0;
  }
  WRNN_REQUIRE(g->out && g->dout && g->dq && !g->dk == !g->dv, "wrnn_attention_backward: null pointer");
  WRNN_REQUIRE(!g->dtable || p.table, "wrnn_attention_backward: a table's gradient without a table");
  const size_t need = wrnn_attention_backward_workspace_bytes(desc);
  WRNN_REQUIRE(workspace && workspace_bytes >= need && !((uintptr_t)workspace & 15),
               "wrnn_attention_backward: workspace of %zu bytes, %zu are needed, on 16 bytes", workspace_bytes, need);
  const int es = desc->dtype == WRNN_FLOAT32 ? 4 : 2;
  struct Rows {
    const void* at;
    const int64_t* stride;
    int64_t *b, *h, *t;
    int heads, len;
  };
  for (const Rows& x : {Rows{p.o_in = g->out, g->out_stride, &p.oi_b, &p.oi_h, &p.oi_t, p.H, p.Tq},
                        Rows{p.dout = g->dout, g->dout_stride, &p.do_b, &p.do_h, &p.do_t, p.H, p.Tq},
                        Rows{p.dq = g->dq, g->dq_stride, &p.dq_b, &p.dq_h, &p.dq_t, p.H, p.Tq},
                        Rows{p.dk = g->dk, g->dk_stride, &p.dk_b, &p.dk_h, &p.dk_t, p.Hkv, p.Tk},
                        Rows{p.dv = g->dv, g->dv_stride, &p.dv_b, &p.dv_h, &p.dv_t, p.Hkv, p.Tk}}) {
    *x.b = attn::stride_of(p.B, x.stride[0]), *x.h = attn::stride_of(x.heads, x.stride[1]), *x.t = attn::stride_of(x.len, x.stride[2]);
    WRNN_REQUIRE(attn::rows_on_four(x.at, *x.b, *x.h, *x.t, es), "wrnn_attention_backward: rows have to start on the bytes of four elements");
  }
  // (of these only dout's rows go through tiles)
  WRNN_REQUIRE(p.do_t >= 0 && p.do_t < attn::kMaxRowStride, "wrnn_attention_backward: position strides of dout are in 0 .. 2^22 - 1 elements");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* w = static_cast<char*>(workspace);
  if (!stats) {  // made anew: the forward kernel without an output
    attn::plan(&p);
    p.stats = reinterpret_cast<float*>(w);
    p.part = reinterpret_cast<float*>(w + attn::stats_bytes(p));
    if (desc->dtype == WRNN_FLOAT32 ? attn::forward<float>(p, st) : attn::forward<__bf16>(p, st)) return 1;
  } else {
    p.stats = const_cast<float*>(stats);
  }
  attn::plan_backward(&p, desc->dtype);
  p.delta = reinterpret_cast<float*>(w += attn::stats_bytes(p));
  p.dtable_part = reinterpret_cast<float*>(w += attn::delta_bytes(p, desc->dtype));
  p.dq_part = reinterpret_cast<float*>(w += attn::table_bytes(p));
  p.dkv_part = reinterpret_cast<float*>(w + attn::dq_bytes(p));
  return desc->dtype == WRNN_FLOAT32 ? attn::backward<float>(p, g->dtable, st) : attn::backward<__bf16>(p, g->dtable, st);
}
