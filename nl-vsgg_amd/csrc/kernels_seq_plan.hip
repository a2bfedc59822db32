// kernels_seq_plan.hip -- how a call of attention over packed sequences is run: the plan, and fp32 tensors as bfloat16 planes.
#include <algorithm>

#include "kernels_seq.h"
#include "seq_attn.h"

namespace sttran {

// x [rows][heads][d] -> planes [rows][heads][3][d padded to 8]: 8 columns a thread; blockIdx.y: which tensor.  Reads 4 bytes an element
// and writes 6, once (four tensors of 8000 rows, 8 heads of 242: 107 us, 6.0 TB/s, some of it out of the caches).  Numbers that the first
// rounding takes to infinity are cut off instead; infinities and NaN stay in the first plane alone.
struct SeqSplitArgs {
  SeqAttnArgs::In in[4];
  char* out[4];
  int64_t rows[4];
  int heads[4], d, aln;
};
__global__ void __launch_bounds__(256) seq_split_kernel(SeqSplitArgs A) {
  const int which = blockIdx.y, heads = A.heads[which], nc = (A.d + 7) / 8;
  const int64_t items = A.rows[which] * heads * nc;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
    const int64_t rh = i / nc, row = rh / heads;
    const int c = (int)(i - rh * nc), head = (int)(rh - row * heads);
    const char* p = A.in[which].p + row * A.in[which].t + head * A.in[which].h;
    seq_u32x4 x[2], pl[3] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
    x[0] = seq_row_chunk(p, 2 * c, 4 * A.d, A.aln);
    x[1] = seq_row_chunk(p, 2 * c + 1, 4 * A.d, A.aln);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = __uint_as_float(x[j >> 2][j & 3]);
      __bf16 hi, mid, lo;
      seq_split3(v, hi, mid, lo);
      if (!(fabsf((float)hi) < INFINITY)) {
        const float cut = __uint_as_float(__float_as_uint(v) & 0xffff0000u), rest = fabsf(v) < INFINITY ? v - cut : 0.f;
        if (v == v) hi = (__bf16)cut;
        mid = (__bf16)rest;
        lo = (__bf16)(rest - (float)mid);
      }
      SeqElt<__bf16>::put(pl[0], j, (float)hi);
      SeqElt<__bf16>::put(pl[1], j, (float)mid);
      SeqElt<__bf16>::put(pl[2], j, (float)lo);
    }
    char* o = A.out[which] + rh * (3 * 16 * nc) + 16 * c;
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<seq_u32x4*>(o + q * 16 * nc) = pl[q];
  }
}

static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// Planes take the matrix products from fp32 instructions to bfloat16 ones (6 of them for one, of a sixteenth of the time each) and cost a
// pass over the tensors, three times the LDS of a tile and up to three more launches.  Measured on 16384 rows, 8 heads, a training step:
//   64 columns: 128 keys 323 us on fp32 instructions, 308 on planes; 256 keys 514, 347; 2048 keys 2317, 1091
//   128: 128 keys 467, 594; 256 keys 729, 736; 512 keys 1181, 943; 2048 keys 3298, 2137
//   200: 512 keys 2151, 2148 (forward alone 474, 602); 1024 keys 3565, 3041 (790, 818); 2048 keys 5957, 4608 (1369, 1228)
// and on calls too small to fill the card (one sequence): 2 heads of 64 columns, 256 rows 158, 106 (26, 24); 2 of 128, 512 rows 178, 137
// (53, 35); 2 of 200, 1024 rows 275, 263 (42, 54).
static bool use_planes(int bf16, const SeqAttnArgs& A) {
  if (bf16 || A.nseq <= 0) return false;
  return A.tk / A.nseq >= (A.d <= 64 ? 256 : A.d <= 128 ? 512 : 1024);
}

// Shares of the keys: where there are too few (row tile, head) pairs for the 256 CUs, up to two workgroups a CU, 256 keys a share at
// least.  The keys that a tile sees are known on the device alone; their number is taken from the tensors' sizes, and a share of
// a shorter range is shorter.  (8 heads, 128 columns, one share and these: 64 rows over 8192 keys 163 -> 25 us in bfloat16, 1053 -> 54 in
// fp32; 1024 rows over 8192 keys 165 -> 78, 519 -> 262; 2 x 16 rows over 512 keys 35 -> 26, 145 -> 82.)
static int fwd_splits(int bf16, bool planes, const SeqAttnArgs& A) {
  const int tile = seq_attn_fwd_tile(bf16, planes, A.d);
  const int64_t wgs = ((int64_t)A.tq + tile - 1) / tile * A.hq;
  if (wgs == 0 || wgs >= 256 || A.nseq <= 0) return 1;
  const int64_t n = std::min<int64_t>((512 + wgs - 1) / wgs, A.tk / A.nseq / 256);
  return (int)std::max<int64_t>(1, std::min<int64_t>(n, 64));
}
// Shares of a key tile's work: none with 1024 workgroups or more (4 a CU: as the order masks, their work differs by up to the whole
// length), else as many as bring it to 1536 (3 x 8000 rows, 8 heads over 2 of 64, 1412 us; to 1024 1502, to 2048 1417), 8 at most, within
// 512 MB of partial sums.  (A training step with one share and these: one
// sequence of 4096 rows, 8 heads, 444 -> 379 us; 6 of 4000, 8 heads over 2, 930 -> 756; three of 6000, 8 over 4, 1498 -> 1340.)  A
// share is 32 tiles at least where every CU has a workgroup anyway: less does not pay for the join (40 of 600 rows, 8 over 4, 364 us in
// one share, 420 in two), 8 where not.
static int dkv_splits(int bf16, bool planes, const SeqAttnArgs& A) {
  const int rb = seq_attn_dkv_tile(bf16, planes, A.d);
  const int64_t wgs = ((int64_t)A.tk + rb - 1) / rb * A.hk, bytes = (int64_t)A.tk * A.hk * A.d * 8;
  if (wgs == 0 || wgs >= 1024) return 1;
  const int64_t work = (int64_t)(A.hq / A.hk) * ((A.tq / (A.nseq > 0 ? A.nseq : 1) + 31) / 32);       // query tiles a key tile sees, about
  int64_t n = std::min<int64_t>((1536 + wgs - 1) / wgs, 8);
  n = std::min<int64_t>(n, work / (wgs >= 256 ? 32 : 8));
  n = std::min<int64_t>(n, (int64_t(512) << 20) / std::max<int64_t>(bytes, 1));
  return (int)std::max<int64_t>(n, 1);
}

SeqAttnPlan seq_attn_plan(int bf16, const SeqAttnArgs& A, bool backward) {
  SeqAttnPlan P{};
  P.planes = use_planes(bf16, A);
  int64_t at = 0;
  const auto take = [&](int64_t n) { const int64_t r = at; at = up256(at + n); return r; };
  if (backward) {
    P.rows = take((int64_t)A.tq * 16);
    P.delta = take((int64_t)A.hq * A.tq * 4);
    P.splits = dkv_splits(bf16, P.planes, A);
    P.part = take(P.splits > 1 ? (int64_t)P.splits * 2 * A.tk * A.hk * A.d * 4 : 0);
  } else {
    P.splits = fwd_splits(bf16, P.planes, A);
    P.part = take(P.splits > 1 ? (int64_t)P.splits * A.hq * A.tq * (A.d + 2) * 4 : 0);
  }
  if (P.planes) {
    const int64_t row = (int64_t)(A.d + 7) / 8 * 48;
    P.plane[0] = take(A.tq * row * A.hq);
    P.plane[1] = take(A.tk * row * A.hk);
    P.plane[2] = take(A.tk * row * A.hk);
    P.plane[3] = backward ? take(A.tq * row * A.hq) : 0;
  }
  P.bytes = at;
  return P;
}

static hipError_t make_planes(hipStream_t s, SeqAttnArgs& A, const SeqAttnPlan& P, char* ws, int tensors) {
  SeqSplitArgs S{};
  int64_t most = 0;
  const int nc = (A.d + 7) / 8;
  for (int i = 0; i < tensors; ++i) {
    const bool q = i == 0 || i == 3;
    S.in[i] = A.raw[i];
    S.out[i] = ws + P.plane[i];
    S.rows[i] = q ? A.tq : A.tk;
    S.heads[i] = q ? A.hq : A.hk;
    most = std::max(most, S.rows[i] * S.heads[i] * nc);
  }
  S.d = A.d; S.aln = A.aln;
  const int64_t blocks = (most + 255) / 256;
  if (blocks > 0) seq_split_kernel<<<dim3((unsigned)std::min<int64_t>(blocks, 8192), (unsigned)tensors), 256, 0, s>>>(S);
  const int64_t h = 48 * (int64_t)nc;
  A.q = S.out[0]; A.k = S.out[1]; A.v = S.out[2]; A.dout = S.out[3];
  A.q_h = A.k_h = A.v_h = A.do_h = h;
  A.q_t = A.do_t = h * A.hq;
  A.k_t = A.v_t = h * A.hk;
  return hipGetLastError();
}

hipError_t launch_seq_attn_forward(hipStream_t s, int bf16, const SeqAttnArgs& args, const SeqAttnPlan& P, char* ws) {
  SeqAttnArgs A = args;
  if (A.tq == 0) return hipSuccess;
  A.splits = P.splits;
  A.part = reinterpret_cast<float*>(ws + P.part);
  if (P.planes) {
    const hipError_t e = make_planes(s, A, P, ws, 3);
    if (e != hipSuccess) return e;
  }
  return launch_seq_attn_fwd(s, bf16, P.planes, A);
}

hipError_t launch_seq_attn_backward(hipStream_t s, int bf16, const SeqAttnArgs& args, const SeqAttnPlan& P, char* ws) {
  SeqAttnArgs A = args;
  A.rows = reinterpret_cast<int4*>(ws + P.rows);
  A.delta = reinterpret_cast<float*>(ws + P.delta);
  A.splits = P.splits;
  A.part = reinterpret_cast<float*>(ws + P.part);
  if (P.planes) {
    const hipError_t e = make_planes(s, A, P, ws, 4);
    if (e != hipSuccess) return e;
  }
  return launch_seq_attn_bwd(s, bf16, P.planes, A);
}

}  // namespace sttran
