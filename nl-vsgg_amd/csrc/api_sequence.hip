// api_sequence.hip -- entry points of the sequence operators (no handle): argument checks, then one launch sequence on the
// caller's stream.
#include <cmath>

#include "../../include/sttran_hip.h"
#include "kernels_seq.h"

using namespace sttran;

namespace {

constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1024, kMaxRowBytes = int64_t(1) << 24, kMaxCacheRowBytes = int64_t(1) << 22;
constexpr int64_t kMaxHeadRows = (int64_t(1) << 29) - 1024;  // a launch over tiles has 8 threads a head's row at most, and fewer than 2^32 of them
constexpr int64_t kMaxCapacity = int64_t(1) << 30;            // rows and a chunk of them are counted in 32 bits
constexpr int32_t kMaxSeq = 1 << 30;                          // the search for a row's sequence adds two numbers of them in 32 bits

bool dtype_ok(int32_t t) { return t == STTRAN_DTYPE_F32 || t == STTRAN_DTYPE_BF16; }
int elt(int32_t t) { return t == STTRAN_DTYPE_BF16 ? 2 : 4; }
bool heads_ok(int32_t hq, int32_t hk, int32_t d) { return hq > 0 && hk > 0 && hq <= 4096 && hq % hk == 0 && d > 0 && d <= 256; }
bool number(float x) { return std::isfinite(x); }
// the kernels work in base 2 and with scale / cap: those have to be numbers too
bool score_ok(float scale, float cap) {
  return number(scale * 1.5f) && number(cap * 3.f) && cap >= 0.f && (cap == 0.f || number(scale / cap * 3.f));
}

// what divides every address and stride that a call touches, up to 16; 0: something is not even aligned to its element
struct Alignment {
  uint64_t bits = 16;
  void at(const void* p) { bits |= reinterpret_cast<uintptr_t>(p); }
  void step(int64_t bytes) { bits |= (uint64_t)bytes; }
  int value(int es) const {
    int a = 16;
    while (bits & (a - 1)) a >>= 1;
    return a < es ? 0 : a;
  }
};

bool row_stride_ok(int64_t s, int es, int64_t most = kMaxRowBytes) { return s >= 0 && s <= most && s * es <= most; }
bool head_stride_ok(int64_t s) { return s >= 0 && s < (int64_t(1) << 40); }

bool workspace_ok(const void* p, int64_t have, int64_t need) { return p && have >= need && !(reinterpret_cast<uintptr_t>(p) & 15); }

hipStream_t str(void* s) { return reinterpret_cast<hipStream_t>(s); }
int code(hipError_t e) { return e == hipSuccess ? STTRAN_OK : STTRAN_ERR_HIP; }

// fills A and checks everything that forward and backward share
bool attention_args(const SttranAttention* a, SeqAttnArgs& A, Alignment& al) {
  if (!a || a->struct_size != sizeof(SttranAttention) || !dtype_ok(a->dtype) || !heads_ok(a->num_q_heads, a->num_kv_heads, a->head_dim))
    return false;
  if (a->num_seq < 0 || a->num_seq > kMaxSeq || a->q_rows < 0 || a->kv_rows < 0 || a->q_rows > kMaxRows || a->kv_rows > kMaxRows) return false;
  if (!score_ok(a->scale, a->score_cap)) return false;
  const int es = elt(a->dtype);
  if (!row_stride_ok(a->q_row_stride, es) || !row_stride_ok(a->k_row_stride, es) || !row_stride_ok(a->v_row_stride, es) ||
      !head_stride_ok(a->q_head_stride) || !head_stride_ok(a->k_head_stride) || !head_stride_ok(a->v_head_stride))
    return false;
  if ((a->q_rows > 0 && !a->q) || (a->kv_rows > 0 && (!a->k || !a->v)) || (a->num_seq > 0 && (!a->seq_off || !a->key_off))) return false;
  if (a->q_rows * a->num_q_heads >= kMaxHeadRows || a->kv_rows * a->num_kv_heads >= kMaxHeadRows) return false;
  A.q = (const char*)a->q; A.k = (const char*)a->k; A.v = (const char*)a->v;
  A.q_t = a->q_row_stride * es; A.q_h = a->q_head_stride * es;
  A.k_t = a->k_row_stride * es; A.k_h = a->k_head_stride * es;
  A.v_t = a->v_row_stride * es; A.v_h = a->v_head_stride * es;
  A.raw[0] = {A.q, A.q_t, A.q_h}; A.raw[1] = {A.k, A.k_t, A.k_h}; A.raw[2] = {A.v, A.v_t, A.v_h};
  A.out = (char*)a->out; A.out_lo = a->dtype == STTRAN_DTYPE_BF16 ? (char*)a->out_residual : nullptr; A.lse = a->lse;
  A.off_q = a->seq_off; A.off_k = a->key_off; A.prefix = a->prefix_len; A.slope = a->distance_slope;
  A.nseq = a->num_seq; A.tq = (int)a->q_rows; A.tk = (int)a->kv_rows;
  A.hq = a->num_q_heads; A.hk = a->num_kv_heads; A.d = a->head_dim; A.causal = a->causal != 0;
  A.cap = a->score_cap; A.scale = a->scale; A.splits = 1;
  al.at(a->q); al.at(a->k); al.at(a->v); al.at(a->out); al.at(A.out_lo);
  al.step(A.q_t); al.step(A.q_h); al.step(A.k_t); al.step(A.k_h); al.step(A.v_t); al.step(A.v_h); al.step((int64_t)A.d * es);
  return true;
}

bool step_args(const SttranAttentionStep* a, SeqStepArgs& A) {
  if (!a || a->struct_size != sizeof(SttranAttentionStep) || !dtype_ok(a->dtype) || !heads_ok(a->num_q_heads, a->num_kv_heads, a->head_dim))
    return false;
  if (a->num_seq < 0 || a->num_seq > 65535 || a->capacity < 0 || a->capacity > kMaxCapacity) return false;
  if (!score_ok(a->scale, a->score_cap)) return false;
  const int es = elt(a->dtype);
  if (!row_stride_ok(a->k_row_stride, es, kMaxCacheRowBytes) || !row_stride_ok(a->v_row_stride, es, kMaxCacheRowBytes) || !head_stride_ok(a->q_seq_stride) ||
      !head_stride_ok(a->q_head_stride) || !head_stride_ok(a->k_seq_stride) || !head_stride_ok(a->k_head_stride) ||
      !head_stride_ok(a->v_seq_stride) || !head_stride_ok(a->v_head_stride))
    return false;
  A.q = (const char*)a->q; A.k = (const char*)a->k; A.v = (const char*)a->v; A.out = (char*)a->out;
  A.q_n = a->q_seq_stride * es; A.q_h = a->q_head_stride * es;
  A.k_n = a->k_seq_stride * es; A.k_t = a->k_row_stride * es; A.k_h = a->k_head_stride * es;
  A.v_n = a->v_seq_stride * es; A.v_t = a->v_row_stride * es; A.v_h = a->v_head_stride * es;
  A.lens = a->lengths; A.slope = a->distance_slope;
  A.n = a->num_seq; A.hq = a->num_q_heads; A.hk = a->num_kv_heads; A.d = a->head_dim; A.capacity = (int)a->capacity;
  A.cap = a->score_cap; A.scale = a->scale;
  A.chunk = seq_step_chunk(A.n, A.hq, A.hk, A.capacity);
  A.splits = A.capacity > 0 ? (A.capacity + A.chunk - 1) / A.chunk : 1;
  return true;
}
int64_t step_workspace(const SeqStepArgs& A) { return A.splits > 1 ? (int64_t)A.splits * A.hq * A.n * (A.d + 2) * 4 : 0; }

bool rotary_args(const SttranRotary* a, SeqRotaryArgs& A, Alignment& al, bool backward) {
  if (!a || a->struct_size != sizeof(SttranRotary) || !dtype_ok(a->dtype)) return false;
  if (a->tokens < 0 || a->tokens > kMaxRows || a->num_q_heads < 0 || a->num_kv_heads < 0 || a->num_q_heads + a->num_kv_heads <= 0 ||
      a->num_q_heads > 4096 || a->num_kv_heads > 4096)
    return false;
  if (a->head_dim <= 0 || a->head_dim > 256 || a->rotary_dim < 0 || a->rotary_dim % 2 || a->rotary_dim > a->head_dim) return false;
  if ((a->q_weight != nullptr) != (a->k_weight != nullptr) || !number(a->eps) || a->eps < 0.f) return false;
  const int es = elt(a->dtype);
  const int64_t row[2] = {a->q_row_stride, a->k_row_stride}, head[2] = {a->q_head_stride, a->k_head_stride};
  const int64_t drow[2] = {a->dq_row_stride, a->dk_row_stride}, dhead[2] = {a->dq_head_stride, a->dk_head_stride};
  const void *x[2] = {a->q, a->k}, *dy[2] = {a->dq_out, a->dk_out};
  void *y[2] = {a->q_out, a->k_out}, *dx[2] = {a->dq, a->dk};
  const int32_t heads[2] = {a->num_q_heads, a->num_kv_heads};
  const float* w[2] = {a->q_weight, a->k_weight};
  float* dw[2] = {a->dq_weight, a->dk_weight};
  al.step((int64_t)a->head_dim * es);
  for (int i = 0; i < 2; ++i) {
    A.heads[i] = heads[i]; A.w[i] = w[i];
    if (heads[i] == 0 || a->tokens == 0) continue;
    const bool reads_x = !backward || w[i];
    if (reads_x) {
      if (!x[i] || !head_stride_ok(row[i]) || !head_stride_ok(head[i])) return false;
      A.x[i] = (const char*)x[i]; A.x_t[i] = row[i] * es; A.x_h[i] = head[i] * es;
      al.at(x[i]); al.step(A.x_t[i]); al.step(A.x_h[i]);
    }
    if (!backward) {
      if (!y[i]) return false;
      A.y[i] = (char*)y[i]; al.at(y[i]);
    } else {
      if (!dy[i] || !dx[i] || !head_stride_ok(drow[i]) || !head_stride_ok(dhead[i])) return false;
      A.dy[i] = (const char*)dy[i]; A.dy_t[i] = drow[i] * es; A.dy_h[i] = dhead[i] * es;
      A.dx[i] = (char*)dx[i];
      al.at(dy[i]); al.at(dx[i]); al.step(A.dy_t[i]); al.step(A.dy_h[i]);
    }
  }
  if (backward && w[0]) { A.dw[0] = dw[0]; A.dw[1] = dw[1]; }
  if (a->tokens > 0 && (!a->positions || (a->rotary_dim > 0 && !a->freq))) return false;
  A.pos = a->positions; A.freq = a->freq; A.tokens = a->tokens; A.d = a->head_dim; A.rot = a->rotary_dim;
  A.interleaved = a->interleaved != 0; A.eps = a->eps;
  return true;
}
int64_t rotary_workspace(const SeqRotaryArgs& A) { return A.w[0] ? (int64_t)seq_rotary_groups(A) * 2 * A.d * 4 + 16 : 0; }

}  // namespace

extern "C" {

int64_t sttran_attention_workspace_bytes(const SttranAttention* args, int32_t backward) {
  SeqAttnArgs A{};
  Alignment al;
  return attention_args(args, A, al) ? seq_attn_plan(args->dtype == STTRAN_DTYPE_BF16, A, backward != 0).bytes : 0;
}

int sttran_attention_forward(const SttranAttention* args, void* stream) {
  SeqAttnArgs A{};
  Alignment al;
  if (!attention_args(args, A, al) || (args->q_rows > 0 && !args->out)) return STTRAN_ERR_INVALID;
  const int bf16 = args->dtype == STTRAN_DTYPE_BF16;
  A.aln = al.value(elt(args->dtype));
  if (!A.aln) return STTRAN_ERR_INVALID;
  const SeqAttnPlan plan = seq_attn_plan(bf16, A, false);
  if (plan.bytes > 0 && !workspace_ok(args->workspace, args->workspace_bytes, plan.bytes)) return STTRAN_ERR_INVALID;
  return code(launch_seq_attn_forward(str(stream), bf16, A, plan, (char*)args->workspace));
}

int sttran_attention_backward(const SttranAttention* args, void* stream) {
  SeqAttnArgs A{};
  Alignment al;
  if (!attention_args(args, A, al)) return STTRAN_ERR_INVALID;
  const int es = elt(args->dtype), bf16 = es == 2;
  if (args->q_rows > 0 && (!args->out || !args->lse || !args->dout || !args->dq)) return STTRAN_ERR_INVALID;
  if (args->kv_rows > 0 && (!args->dk || !args->dv)) return STTRAN_ERR_INVALID;
  if (!row_stride_ok(args->dout_row_stride, es) || !head_stride_ok(args->dout_head_stride)) return STTRAN_ERR_INVALID;
  const SeqAttnPlan plan = seq_attn_plan(bf16, A, true);
  if (plan.bytes > 0 && !workspace_ok(args->workspace, args->workspace_bytes, plan.bytes)) return STTRAN_ERR_INVALID;
  A.dout = (const char*)args->dout;
  A.do_t = args->dout_row_stride * es; A.do_h = args->dout_head_stride * es;
  A.raw[3] = {A.dout, A.do_t, A.do_h};
  A.dq = (char*)args->dq; A.dk = (char*)args->dk; A.dv = (char*)args->dv;
  al.at(A.dout); al.at(A.dq); al.at(A.dk); al.at(A.dv); al.step(A.do_t); al.step(A.do_h);
  A.aln = al.value(es);
  if (!A.aln) return STTRAN_ERR_INVALID;
  return code(launch_seq_attn_backward(str(stream), bf16, A, plan, (char*)args->workspace));
}

int64_t sttran_attention_step_workspace_bytes(const SttranAttentionStep* args) {
  SeqStepArgs A{};
  return step_args(args, A) ? step_workspace(A) : 0;
}

int sttran_attention_step(const SttranAttentionStep* args, void* stream) {
  SeqStepArgs A{};
  if (!step_args(args, A)) return STTRAN_ERR_INVALID;
  if (A.n > 0 && (!A.q || !A.out || !A.lens || (A.capacity > 0 && (!A.k || !A.v)))) return STTRAN_ERR_INVALID;
  Alignment al;
  al.at(A.q); al.at(A.k); al.at(A.v);
  for (int64_t b : {A.q_n, A.q_h, A.k_n, A.k_t, A.k_h, A.v_n, A.v_t, A.v_h, (int64_t)A.d * elt(args->dtype)}) al.step(b);
  A.aln = al.value(elt(args->dtype));
  if (!A.aln) return STTRAN_ERR_INVALID;
  const int64_t need = step_workspace(A);
  if (need > 0 && !workspace_ok(args->workspace, args->workspace_bytes, need)) return STTRAN_ERR_INVALID;
  A.part = (float*)args->workspace;
  return code(launch_seq_step(str(stream), args->dtype == STTRAN_DTYPE_BF16, A));
}

int64_t sttran_rotary_workspace_bytes(const SttranRotary* args) {
  if (!args || args->struct_size != sizeof(SttranRotary) || args->tokens < 0 || args->head_dim <= 0 || args->head_dim > 256) return 0;
  SeqRotaryArgs A{};
  A.tokens = args->tokens; A.d = args->head_dim; A.w[0] = args->q_weight;
  return rotary_workspace(A);
}

int sttran_rotary_forward(const SttranRotary* args, void* stream) {
  SeqRotaryArgs A{};
  Alignment al;
  if (!rotary_args(args, A, al, false)) return STTRAN_ERR_INVALID;
  A.aln = al.value(elt(args->dtype));
  if (!A.aln) return STTRAN_ERR_INVALID;
  return code(launch_seq_rotary_forward(str(stream), args->dtype == STTRAN_DTYPE_BF16, A));
}

int sttran_rotary_backward(const SttranRotary* args, void* stream) {
  SeqRotaryArgs A{};
  Alignment al;
  if (!rotary_args(args, A, al, true)) return STTRAN_ERR_INVALID;
  A.aln = al.value(elt(args->dtype));
  if (!A.aln) return STTRAN_ERR_INVALID;
  if (A.dw[0] || A.dw[1]) {
    if (!workspace_ok(args->workspace, args->workspace_bytes, rotary_workspace(A))) return STTRAN_ERR_INVALID;
    A.part = (float*)args->workspace;
  }
  return code(launch_seq_rotary_backward(str(stream), args->dtype == STTRAN_DTYPE_BF16, A));
}

int sttran_dropout_add(const void* x, const void* residual, void* y, int64_t n, int32_t dtype, double p, const int64_t* rng_state,
                       int64_t key, int64_t offset, int64_t* used, void* stream) {
  if (!dtype_ok(dtype) || n < 0 || n > (int64_t(1) << 46) || !(p >= 0. && p < 1.) || (n > 0 && (!x || !y))) return STTRAN_ERR_INVALID;
  SeqDropoutArgs A{};
  Alignment al;
  al.at(x); al.at(y); al.at(residual);
  A.aln = al.value(elt(dtype));
  if (!A.aln) return STTRAN_ERR_INVALID;
  const double words = std::nearbyint(p * 4294967296.0);
  A.x = (const char*)x; A.res = (const char*)residual; A.y = (char*)y;
  A.rng = rng_state; A.key = key; A.offset = offset; A.used = used; A.n = n;
  A.none = words >= 4294967296.0;                          // below 2^32 are all words
  A.threshold = A.none ? 0u : (uint32_t)words;
  A.mul = (float)(1.0 / (1.0 - p));
  return code(launch_seq_dropout(str(stream), dtype == STTRAN_DTYPE_BF16, A));
}

}  // extern "C"
