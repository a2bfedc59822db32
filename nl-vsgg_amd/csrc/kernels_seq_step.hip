// kernels_seq_step.hip -- attention of ONE new token a sequence over its cached keys and values.
//   o = sum_j p_j v_j over the sequence's live cache rows j < length;  p, z as in kernels_seq_attn.hip with the new token at
//   place length - 1 (its own key is the cache's newest row).
// Bound by reading the cache: every live row of k and v once.  A workgroup takes `chunk` rows of one (sequence, key head) for up
// to GT of the query heads that share it, so shared heads do not read the cache again; several chunks of a sequence are joined
// by a second launch.  LPK lanes hold one row (16 bytes each), every lane group runs its own softmax (maximum, sum, output in
// fp32) over its rows, and the groups are merged once at the end: no communication inside the loop but the dot products.
// Measured: 48 caches of 700 .. 8192 rows, 32 heads over 8 of 128 columns, capped, distances, bfloat16: 172 us, 5.2 TB/s, and 7 us to join;
// one of 2201 rows, 8 heads of 242, fp32: 9 and 5 us.
#include <algorithm>

#include "kernels_seq.h"
#include "seq_attn.h"

namespace sttran {

// Scores of U rows times GT heads are NS = 8 or 16 sums over the LPK lanes of a row.  They are not summed into every lane: at each
// step of the reduction a lane hands half of its sums to the lane across and keeps the other half, so lane i ends with score i
// mod NS alone, and bends, biases and exponentiates that one.  A broadcast within the row of 16 lanes gives each probability back.
// (All lanes on all scores: 283 us where this takes 172 on 48 caches of 700 .. 8192 rows, 32 heads over 8, 128 columns.)
template <int LPK, int GT>
struct SeqStepShape {
  static constexpr int NS = LPK >= 16 && GT > 1 ? 16 : 8, U = NS / GT, KPW = 64 / LPK, NW = 4, STEP = NW * KPW * U;
};
template <int N, int CTRL>                                    // x[0 .. N) -> x[0 .. N / 2): a lane with `up` keeps the upper half
__device__ __forceinline__ void seq_fold(float (&x)[16], bool up) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float keep = up ? x[i + N / 2] : x[i], give = up ? x[i] : x[i + N / 2];
    x[i] = keep + seq_dpp<CTRL>(give);
  }
}
// f over the lanes of the row group that hold the same head (index mod GT)
template <int LPK, int GT, class F>
__device__ __forceinline__ float seq_same_head(float x, F f) {
  if constexpr (LPK == 8) {
#pragma unroll
    for (int o = GT; o < 8; o <<= 1) x = f(x, __shfl_xor(x, o));
  } else {
    if constexpr (GT <= 1) x = f(x, seq_ror<1>(x));
    if constexpr (GT <= 2) x = f(x, seq_ror<2>(x));
    if constexpr (GT <= 4) x = f(x, seq_ror<4>(x));
    x = f(x, seq_ror<8>(x));
  }
  return x;
}
template <int LPK, int I>
__device__ __forceinline__ float seq_score_of(float x) {       // score I of this lane's row group
  if constexpr (LPK == 8) {
    const float a = seq_bcast<I>(x), b = seq_bcast<I + 8>(x);
    return threadIdx.x & 8 ? b : a;
  } else {
    return seq_bcast<I>(x);
  }
}
template <int LPK, int N, int I = 0>
__device__ __forceinline__ void seq_scores_of(float x, float (&out)[16]) {
  if constexpr (I < N) {
    out[I] = seq_score_of<LPK, I>(x);
    seq_scores_of<LPK, N, I + 1>(x, out);
  }
}

template <class T, int LPK, int GT>
__global__ void __launch_bounds__(256) seq_step_kernel(SeqStepArgs A) {
  using S = SeqStepShape<LPK, GT>;
  constexpr int EPL = SeqElt<T>::kPer16, KPW = S::KPW, NW = S::NW, U = S::U, NS = S::NS;
  __shared__ float sm[NW * GT * LPK * EPL + 2 * NW * GT];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane % LPK, kg = lane / LPK;
  const int grp = A.hq / A.hk, gts = (grp + GT - 1) / GT;
  const int kvh = blockIdx.y / gts, g0 = blockIdx.y % gts * GT, n = blockIdx.z;
  const int len = min(max(A.lens[n], 0), A.capacity);
  const int beg = blockIdx.x * A.chunk, end = min(len, beg + A.chunk);
  if (beg >= end && blockIdx.x > 0) return;                 // nothing here (the join knows how many chunks a length fills)
  const int dbytes = A.d * (int)sizeof(T), valid = dbytes - 16 * c;
  const float mul = A.cap > 0.f ? A.scale / A.cap : A.scale * kSeqLog2e, capl = A.cap * kSeqLog2e;

  const int mine = lane & (NS - 1), my_u = mine / GT, my_g = mine % GT;     // the score that this lane finishes
  float q[GT][EPL], acc[GT][EPL], m = -INFINITY, l = 0.f;
  const float slope = A.slope && g0 + my_g < grp ? A.slope[kvh * grp + g0 + my_g] * kSeqLog2e : 0.f;
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    const int head = kvh * grp + g0 + g;
    const seq_u32x4 r = seq_load16(A.q + n * A.q_n + head * A.q_h + 16 * c, g0 + g < grp ? valid : 0, A.aln);
#pragma unroll
    for (int i = 0; i < EPL; ++i) { q[g][i] = SeqElt<T>::get(r, i); acc[g][i] = 0.f; }
  }
  const char *kp = A.k + n * A.k_n + kvh * A.k_h, *vp = A.v + n * A.v_n + kvh * A.v_h;
  const uint32_t k_at = 16 * c < dbytes ? (w * KPW + kg) * (uint32_t)A.k_t + 16 * c : kSeqOob;
  const uint32_t v_at = 16 * c < dbytes ? (w * KPW + kg) * (uint32_t)A.v_t + 16 * c : kSeqOob;
  const seq_u32x4 mask = seq_chunk_mask(c, dbytes);
  for (int k0 = beg; k0 < end; k0 += S::STEP) {
    seq_u32x4 kr[U], vr[U];
    if (A.aln >= 4) {                                       // buffer loads: rows from `end` on are zeros
      const auto rk = seq_rsrc(kp + (int64_t)k0 * A.k_t, A.k_t, end - k0 < S::STEP ? end - k0 : S::STEP, dbytes);
      const auto rv = seq_rsrc(vp + (int64_t)k0 * A.v_t, A.v_t, end - k0 < S::STEP ? end - k0 : S::STEP, dbytes);
#pragma unroll
      for (int u = 0; u < U; ++u)
        kr[u] = __builtin_bit_cast(seq_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_at, u * NW * KPW * (uint32_t)A.k_t, 0));
#pragma unroll
      for (int u = 0; u < U; ++u)
        vr[u] = __builtin_bit_cast(seq_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, v_at, u * NW * KPW * (uint32_t)A.v_t, 0));
      if (dbytes & 15) {                                    // what the last chunk reads behind the row must not meet q's zeros
#pragma unroll
        for (int u = 0; u < U; ++u) kr[u] &= mask;
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = k0 + (u * NW + w) * KPW + kg;
        kr[u] = seq_load16(kp + key * A.k_t + 16 * c, key < end ? valid : 0, A.aln);
        vr[u] = seq_load16(vp + key * A.v_t + 16 * c, key < end ? valid : 0, A.aln);
      }
    }
    float x[16];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) s = fmaf(q[g][i], SeqElt<T>::get(kr[u], i), s);
        x[u * GT + g] = s;
      }
    }
    if constexpr (NS == 16) seq_fold<16, kDppXor15>(x, lane & 8);
    seq_fold<8, kDppXor7>(x, lane & 4);
    seq_fold<4, kDppXor3>(x, lane & 2);
    seq_fold<2, kDppXor1>(x, lane & 1);
    float s = x[0];
    if constexpr (LPK >= 16 && NS == 8) s += seq_ror<8>(s);
    if constexpr (LPK >= 32) s = seq_add16(s);
    if constexpr (LPK >= 64) s = seq_add32(s);
    const int key = k0 + (my_u * NW + w) * KPW + kg;
    s *= mul;
    if (A.cap > 0.f) s = capl * seq_tanh<false>(s);
    s = key < end ? fmaf(-slope, (float)(len - 1 - key), s) : -INFINITY;
    const float mn = fmaxf(m, seq_same_head<LPK, GT>(s, [](float a, float b) { return fmaxf(a, b); }));
    const float ms = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - ms), p = __builtin_amdgcn_exp2f(s - ms);
    m = mn; l = fmaf(l, al, p);
    float ps[16], as[16];
    seq_scores_of<LPK, NS>(p, ps);
    seq_scores_of<LPK, GT>(al, as);
#pragma unroll
    for (int g = 0; g < GT; ++g) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[g][i] *= as[g];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < EPL; ++i) acc[g][i] = fmaf(ps[u * GT + g], SeqElt<T>::get(vr[u], i), acc[g][i]);
    }
  }
  l = seq_same_head<LPK, GT>(l, [](float a, float b) { return a + b; });
  // one score lane a row group would count twice where NS < 16 lanes hold it: the sum above went round the row of 16
  if constexpr (LPK >= 16 && NS == 8) l *= 0.5f;
  float mg[16], lg[16];
  seq_scores_of<LPK, GT>(m, mg);
  seq_scores_of<LPK, GT>(l, lg);
  // merge the lane groups of the wave, then the waves
#pragma unroll
  for (int g = 0; g < GT; ++g) {
#pragma unroll
    for (int o = LPK; o < 64; o <<= 1) {
      const float mo = __shfl_xor(mg[g], o), lo = __shfl_xor(lg[g], o), mn = fmaxf(mg[g], mo), ms = mn == -INFINITY ? 0.f : mn;
      const float a = __builtin_amdgcn_exp2f(mg[g] - ms), b = __builtin_amdgcn_exp2f(mo - ms);
      lg[g] = lg[g] * a + lo * b;
      mg[g] = mn;
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[g][i] = acc[g][i] * a + __shfl_xor(acc[g][i], o) * b;
    }
  }
  float* stat = sm + NW * GT * LPK * EPL;
  if (kg == 0) {
#pragma unroll
    for (int g = 0; g < GT; ++g) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) sm[((w * GT + g) * LPK + c) * EPL + i] = acc[g][i];
      if (c == 0) { stat[(w * GT + g) * 2] = mg[g]; stat[(w * GT + g) * 2 + 1] = lg[g]; }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < GT * LPK * EPL; i += 256) {
    const int g = i / (LPK * EPL), col = i % (LPK * EPL), head = kvh * grp + g0 + g;
    if (g0 + g >= grp || col >= A.d) continue;
    float mn = -INFINITY, ls = 0.f, o = 0.f;
#pragma unroll
    for (int y = 0; y < NW; ++y) mn = fmaxf(mn, stat[(y * GT + g) * 2]);
    const float ms = mn == -INFINITY ? 0.f : mn;
#pragma unroll
    for (int y = 0; y < NW; ++y) {
      const float f = __builtin_amdgcn_exp2f(stat[(y * GT + g) * 2] - ms);
      ls = fmaf(stat[(y * GT + g) * 2 + 1], f, ls);
      o = fmaf(sm[(y * GT + g) * LPK * EPL + col], f, o);
    }
    if (A.splits > 1) {
      const int64_t at = ((int64_t)blockIdx.x * A.hq + head) * A.n + n;
      A.part[at * A.d + col] = o;
      if (col == 0) {
        float* ps = A.part + (int64_t)A.splits * A.hq * A.n * A.d + at * 2;
        ps[0] = mn; ps[1] = ls;
      }
    } else {
      const float y = ls == 0.f ? 0.f : o / ls;
      const int64_t at = ((int64_t)n * A.hq + head) * A.d + col;
      if constexpr (sizeof(T) == 4) reinterpret_cast<float*>(A.out)[at] = y;
      else reinterpret_cast<uint16_t*>(A.out)[at] = (uint16_t)SeqElt<T>::bits(y);
    }
  }
}

template <class T, int LPK>
static hipError_t step_g(hipStream_t s, const SeqStepArgs& A) {
  const int grp = A.hq / A.hk;
  const auto grid = [&](int gt) { return dim3((unsigned)A.splits, (unsigned)(A.hk * ((grp + gt - 1) / gt)), (unsigned)A.n); };
  if (grp == 1) seq_step_kernel<T, LPK, 1><<<grid(1), 256, 0, s>>>(A);
  else if (grp == 2) seq_step_kernel<T, LPK, 2><<<grid(2), 256, 0, s>>>(A);
  else if (grp <= 4) seq_step_kernel<T, LPK, 4><<<grid(4), 256, 0, s>>>(A);
  else seq_step_kernel<T, LPK, 8><<<grid(8), 256, 0, s>>>(A);
  return hipGetLastError();
}
template <class T>
static hipError_t step(hipStream_t s, const SeqStepArgs& A) {
  const int chunks = (A.d * (int)sizeof(T) + 15) / 16;
  if (chunks <= 8) return step_g<T, 8>(s, A);
  if (chunks <= 16) return step_g<T, 16>(s, A);
  if constexpr (sizeof(T) == 4)
    if (chunks > 32) return step_g<T, 64>(s, A);
  return step_g<T, 32>(s, A);
}

// rows of the cache that one workgroup takes: about 4096 workgroups at full length (lengths differ, and a CU holds several), 192 rows at
// least.  Measured, with the join: 48 caches of 900 .. 8192 rows, 32 heads over 8 of 128 columns, 186 us (190 at 8192 workgroups, 239 at
// 32768); one of 16000 rows 24.5 (33.0 at 64 rows, 21.8 at 256), 100 of 56 .. 512 rows, 8 of 64, 17.4 (32.9, 17.5), one of 2240 rows, 8 of
// 242 in fp32, 13.1 (13.1, 14.4)
int seq_step_chunk(int n, int hq, int hk, int capacity) {
  const int grp = hq / hk, gt = grp <= 1 ? 1 : grp <= 2 ? 2 : grp <= 4 ? 4 : 8;
  const int64_t per = (int64_t)n * hk * ((grp + gt - 1) / gt);
  const int64_t want = (per * capacity + 4095) / 4096;
  const int64_t chunk = std::min<int64_t>((want + 63) / 64 * 64, capacity);       // one cache for thousands of sequences: `want` passes 32 bits
  return (int)std::max<int64_t>(chunk, 192);
}

hipError_t launch_seq_step(hipStream_t s, int bf16, const SeqStepArgs& A) {
  if (A.n == 0) return hipSuccess;
  hipError_t e = bf16 ? step<__bf16>(s, A) : step<float>(s, A);
  if (e != hipSuccess || A.splits == 1) return e;
  SeqAttnArgs J{};
  J.out = A.out; J.part = A.part; J.tq = A.n; J.hq = A.hq; J.d = A.d; J.splits = A.splits;
  return launch_seq_attn_join(s, bf16, J, A.lens, A.chunk, A.capacity);
}

}  // namespace sttran
