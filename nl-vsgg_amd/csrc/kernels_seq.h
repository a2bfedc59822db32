// kernels_seq.h -- launch interface of the sequence operators (kernels_seq_*.hip).  Internal to libsttran_hip.so.
#pragma once
#include "kernels.h"
#include "seq_common.h"

namespace sttran {

// ---- attention over packed sequences
// How a call is run, from what the host knows, and where things lie in its workspace (byte offsets)
struct SeqAttnPlan {
  bool planes;               // fp32 as three bfloat16 planes
  int splits;                // shares of the keys (forward) or of a key tile's work (backward); 1: none
  int64_t rows, delta, part, plane[4], bytes;
};
SeqAttnPlan seq_attn_plan(int bf16, const SeqAttnArgs& A, bool backward);
hipError_t launch_seq_attn_forward(hipStream_t s, int bf16, const SeqAttnArgs& A, const SeqAttnPlan& P, char* workspace);
hipError_t launch_seq_attn_backward(hipStream_t s, int bf16, const SeqAttnArgs& A, const SeqAttnPlan& P, char* workspace);
// their parts: the launches themselves, planes already made; own rows of a forward / key tile workgroup
hipError_t launch_seq_attn_fwd(hipStream_t s, int bf16, bool planes, const SeqAttnArgs& A);
hipError_t launch_seq_attn_bwd(hipStream_t s, int bf16, bool planes, const SeqAttnArgs& A);
int seq_attn_fwd_tile(int bf16, bool planes, int d);
int seq_attn_dkv_tile(int bf16, bool planes, int d);
// joins partial outputs [split][head][row][d] + [split][head][row][2].  lens (device, per row) and chunk: only the shares that a
// row's length fills were written (lens == nullptr: all of them)
hipError_t launch_seq_attn_join(hipStream_t s, int bf16, const SeqAttnArgs& A, const int* lens, int chunk, int capacity);

// ---- one new token a sequence over its cache (strides in BYTES)
struct SeqStepArgs {
  const char *q, *k, *v;
  int64_t q_n, q_h, k_n, k_t, k_h, v_n, v_t, v_h;
  char* out;                       // contiguous [n, q heads, d]
  const int* lens;
  const float* slope;
  float* part;
  int n, hq, hk, d, capacity, chunk, splits, aln;
  float cap, scale;
};
int seq_step_chunk(int n, int hq, int hk, int capacity);
hipError_t launch_seq_step(hipStream_t s, int bf16, const SeqStepArgs& A);

// ---- per-head norm and rotary positions of queries and keys (strides in BYTES; outputs and gradients contiguous)
struct SeqRotaryArgs {
  const char *x[2], *dy[2];        // q, k: [tokens, heads, d]; backward: gradients of the outputs
  int64_t x_t[2], x_h[2], dy_t[2], dy_h[2];
  char *y[2], *dx[2];
  const float* w[2];               // [d] norm weights, or null: no norm
  float* dw[2];
  float* part;                     // partial weight gradients [workgroups][2][d]
  const int64_t* pos;
  const float* freq;               // [rot / 2] angle a position step
  int64_t tokens;
  int heads[2], d, rot, interleaved, aln;
  uint32_t per_head;               // the launch's own
  float eps;
};
int seq_rotary_groups(const SeqRotaryArgs& A);          // workgroups of a backward launch
hipError_t launch_seq_rotary_forward(hipStream_t s, int bf16, const SeqRotaryArgs& A);
hipError_t launch_seq_rotary_backward(hipStream_t s, int bf16, const SeqRotaryArgs& A);

// ---- dropout with the residual sum
struct SeqDropoutArgs {
  const char *x, *res;
  char* y;
  const int64_t* rng;              // device: {key, first counter}; null: the two values below
  int64_t key, offset;
  int64_t* used;                   // optional, device: the state this launch drew from
  int64_t n;
  uint32_t threshold;              // words below it drop their element
  bool none;                       // every element is dropped
  float mul;
  int aln;
};
hipError_t launch_seq_dropout(hipStream_t s, int bf16, const SeqDropoutArgs& A);

}  // namespace sttran
