// seq_common.h -- device helpers of the sequence operators (kernels_seq_*.hip): element types, row loads that respect any
// alignment of two bytes or more, and the launch arguments.  Internal to libsttran_hip.so.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sttran {

typedef float seq_f32x16 __attribute__((ext_vector_type(16)));
typedef float seq_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 seq_bf16x8 __attribute__((ext_vector_type(8)));
typedef short seq_s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t seq_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t seq_u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));   // 16 bytes at any multiple of 4

constexpr float kSeqLog2e = 1.4426950408889634f;

// 16 bytes from `p`, the bytes from `valid` on as zeros.  `aln`: a power of two (2 .. 16) that divides the address and every
// row's length, so no piece straddles the row's end.  A vector load needs no more than dword alignment on this card.
__device__ __forceinline__ seq_u32x4 seq_load16(const char* p, int valid, int aln) {
  if (valid >= 16 && aln >= 4) return *reinterpret_cast<const seq_u32x4_a4*>(p);
  seq_u32x4 r = {0, 0, 0, 0};
  if (valid <= 0) return r;
  if (aln >= 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * i < valid) r[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (2 * i < valid) r[i >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p + 2 * i) << (16 * (i & 1));
  }
  return r;
}

// chunk c of a row at `row`, what lies behind the row's dbytes as zeros, without branches between lanes (a divergent tail makes
// every load of a loop wait by itself): chunks at the row's end read its last 16 bytes and shift them (selects alone: the same as
// an if / else if chain over the tail's length has been compiled to a path that skips one of them)
__device__ __forceinline__ seq_u32x4 seq_row_chunk(const char* row, int c, int dbytes, int aln) {
  if (aln < 4 || dbytes < 16) return seq_load16(row + 16 * c, dbytes - 16 * c, aln);
  const int at = min(16 * c, dbytes - 16), skip = (16 * c - at) >> 2;          // dwords of it that lie before the chunk
  const seq_u32x4 r = *reinterpret_cast<const seq_u32x4_a4*>(row + at);
  if ((dbytes & 15) == 0 && dbytes >= 16 * 64) return r;
  const bool s1 = skip == 1, s2 = skip == 2, s3 = skip == 3, s0 = skip == 0;
  seq_u32x4 x;
  x[0] = s0 ? r[0] : s1 ? r[1] : s2 ? r[2] : s3 ? r[3] : 0u;
  x[1] = s0 ? r[1] : s1 ? r[2] : s2 ? r[3] : 0u;
  x[2] = s0 ? r[2] : s1 ? r[3] : 0u;
  x[3] = s0 ? r[3] : 0u;
  return x;
}

__device__ __forceinline__ void seq_store16(char* p, seq_u32x4 r, int valid, int aln) {
  if (valid >= 16 && aln >= 4) {
    *reinterpret_cast<seq_u32x4_a4*>(p) = r;
  } else if (aln >= 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * i < valid) *reinterpret_cast<uint32_t*>(p + 4 * i) = r[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (2 * i < valid) *reinterpret_cast<uint16_t*>(p + 2 * i) = (uint16_t)(r[i >> 1] >> (16 * (i & 1)));
  }
}

// fp32 <-> the stored type; rounding to bfloat16 is to nearest, ties to even (half a step: 2^-8 of the
// value at most)
template <class T> struct SeqElt;
template <> struct SeqElt<float> {
  static constexpr int kPer16 = 4;
  static __device__ __forceinline__ float get(const seq_u32x4& r, int i) { return __uint_as_float(r[i]); }
  static __device__ __forceinline__ void put(seq_u32x4& r, int i, float x) { r[i] = __float_as_uint(x); }
  static __device__ __forceinline__ float at(const char* p) { return *reinterpret_cast<const float*>(p); }
  static __device__ __forceinline__ float round(float x) { return x; }
};
template <> struct SeqElt<__bf16> {
  static constexpr int kPer16 = 8;
  static __device__ __forceinline__ float get(const seq_u32x4& r, int i) {
    return __uint_as_float((i & 1) ? (r[i >> 1] & 0xffff0000u) : (r[i >> 1] << 16));
  }
  static __device__ __forceinline__ uint32_t bits(float x) { return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x); }
  static __device__ __forceinline__ void put(seq_u32x4& r, int i, float x) {          // r starts as zeros
    r[i >> 1] |= bits(x) << (16 * (i & 1));
  }
  static __device__ __forceinline__ float at(const char* p) {
    return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
  }
  static __device__ __forceinline__ float round(float x) { return (float)(__bf16)x; }
};

// ---- lane exchanges without LDS traffic (DPP: within rows of 16 lanes; permlane swaps: between rows)
template <int CTRL>
__device__ __forceinline__ float seq_dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
constexpr int kDppXor1 = 0xB1, kDppXor3 = 0x1B, kDppXor7 = 0x141, kDppXor15 = 0x140;    // quad_perm, row_half_mirror, row_mirror
template <int N> __device__ __forceinline__ float seq_ror(float x) { return seq_dpp<0x120 + N>(x); }         // lane i from i - N of 16
template <int N> __device__ __forceinline__ float seq_bcast(float x) { return seq_dpp<0x150 + N>(x); }       // lane N of the row
__device__ __forceinline__ float seq_add16(float x) {                                                        // x + lane ^ 16
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float seq_add32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// sum over groups of N lanes, the same bits in each of them
template <int N>
__device__ __forceinline__ float seq_group_sum(float x) {
  x += seq_dpp<kDppXor1>(x);
  if constexpr (N > 2) x += seq_dpp<kDppXor3>(x);
  if constexpr (N > 4) x += seq_dpp<kDppXor7>(x);
  if constexpr (N > 8) x += seq_dpp<kDppXor15>(x);
  if constexpr (N > 16) x = seq_add16(x);
  if constexpr (N > 32) x = seq_add32(x);
  return x;
}

// ---- attention over packed sequences: arguments of the launches (strides in BYTES) ---------------------------------------
struct SeqAttnArgs {
  const char *q, *k, *v, *dout;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, do_t, do_h;
  struct In { const char* p; int64_t t, h; } raw[4];      // q, k, v, dout as the caller gave them (the above may be planes of them)
  char *out, *out_lo, *dq, *dk, *dv;      // contiguous [rows, heads, d]; out_lo: what rounding took from out (bfloat16, training)
  float* lse;                             // [q heads][q rows], base 2: max + log2(sum); +inf for a row that sees nothing
  float* delta;                           // [q heads][q rows]: sum of dout * out
  int4* rows;                             // [q rows]: first key row, end of its key rows, key row at distance zero
  float* part;                            // partial outputs of a launch that is split over the keys
  const int *off_q, *off_k, *prefix;
  const float* slope;
  int nseq, tq, tk, hq, hk, d, causal, aln, splits;
  float cap, scale;
};

// The key rows [lo, hi) that query row t sees, and the key row at distance zero from it.  Every mask here (documents, order,
// prefix) leaves one contiguous range: keys below max(position + 1, prefix) of the row's own sequence.  Offsets are device data
// that the host cannot check without waiting: they are clamped to the tensors, so wrong ones give wrong rows, never a fault.
struct SeqRow { int lo, hi, base; };
__device__ __forceinline__ int seq_find(const int* off, int n, int t) {      // first s with off[s + 1] > t (n if none)
  int a = 0, b = n;
  while (a < b) {
    const int m = (a + b) >> 1;
    if (off[m + 1] > t) b = m; else a = m + 1;
  }
  return a;
}
// the same for a t that the wave shares, 64 offsets at a time: two dependent loads for 4096 sequences instead of twelve
__device__ __forceinline__ int seq_find_wave(const int* off, int n, int t) {
  const int lane = threadIdx.x & 63;
  int a = 0, b = n;
  while (a < b) {                                         // the answer is one of a .. b
    const int step = (b - a + 63) >> 6, at = a + (lane + 1) * step - 1;
    const uint64_t yes = __ballot(at >= b || off[at + 1] > t);
    a += (yes ? __builtin_ctzll(yes) : 64) * step;
    b = min(a + step - 1, b);
    a = min(a, b);
  }
  return a;
}
__device__ __forceinline__ SeqRow seq_row(const SeqAttnArgs& A, int t, int s) {         // s: seq_find of t
  SeqRow r{0, 0, 0};
  if (t >= A.tq || s >= A.nseq) return r;
  const int q0 = A.off_q[s], q1 = A.off_q[s + 1];
  if (t < q0) return r;
  const int k0 = min(max(A.off_k[s], 0), A.tk), k1 = min(max(A.off_k[s + 1], k0), A.tk);
  const int pos = (t - q0) + (k1 - k0) - (q1 - q0);
  int len = k1 - k0;
  if (A.causal) len = min(len, max(max(pos + 1, A.prefix ? A.prefix[s] : 0), 0));
  r.lo = k0; r.hi = k0 + len; r.base = k0 + pos;
  if (len <= 0) r.lo = r.hi = 0;
  return r;
}
// row t of the 32 from row0 on that a wave holds
__device__ __forceinline__ SeqRow seq_row_of_wave(const SeqAttnArgs& A, int row0, int t) {
  const int s0 = seq_find_wave(A.off_q, A.nseq, row0), at = s0 + 1 + (threadIdx.x & 63);
  const int o = at <= A.nseq ? A.off_q[at] : 0x7fffffff;
  const int ends = __popcll(__ballot(o <= row0 + 31));    // sequences that end within these rows
  int s = s0;
  if (ends == 64) s = seq_find(A.off_q, A.nseq, t);
  else
    for (int j = 0; j < ends; ++j) s += __builtin_amdgcn_readlane(o, j) <= t;
  return seq_row(A, t, s);
}

}  // namespace sttran
