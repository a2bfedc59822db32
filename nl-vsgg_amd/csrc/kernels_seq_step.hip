// kernels_seq_step.hip -- attention of ONE new token a sequence over its cached keys and values.
//   o = sum_j p_j v_j over the sequence's live cache rows j < length;  p, z as in kernels_seq_attn.hip with the new token at
//   place length - 1 (its own key is the cache's newest row).
// Bound by reading the cache: every live row of k and v once.  A workgroup takes `chunk` rows of one (sequence, key head) for up
// to GT of the query heads that share it, so shared heads do not read the cache again; several chunks of a sequence are joined
// by a second launch.  LPK lanes hold one row (16 bytes each), every lane group runs its own softmax (maximum, sum, output in
// fp32) over its rows, and the groups are merged once at the end: no communication inside the loop but the dot products.
#include "kernels_seq.h"

namespace sttran {

template <class T, int LPK, int GT>
__global__ void __launch_bounds__(256) seq_step_kernel(SeqStepArgs A) {
  constexpr int EPL = SeqElt<T>::kPer16, KPW = 64 / LPK, NW = 4, U = GT >= 8 ? 2 : 4, STEP = NW * KPW * U;
  __shared__ float sm[NW * GT * LPK * EPL + 2 * NW * GT];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane % LPK, kg = lane / LPK;
  const int grp = A.hq / A.hk, gts = (grp + GT - 1) / GT;
  const int kvh = blockIdx.y / gts, g0 = blockIdx.y % gts * GT, n = blockIdx.z;
  const int len = min(max(A.lens[n], 0), A.capacity);
  const int beg = blockIdx.x * A.chunk, end = min(len, beg + A.chunk);
  if (beg >= end && blockIdx.x > 0) return;                 // nothing here (the join knows how many chunks a length fills)
  const int dbytes = A.d * (int)sizeof(T), valid = dbytes - 16 * c;
  const float mul = A.cap > 0.f ? A.scale / A.cap : A.scale * kSeqLog2e, capl = A.cap * kSeqLog2e;

  float q[GT][EPL], acc[GT][EPL], m[GT], l[GT], sl[GT];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    const int head = kvh * grp + g0 + g;
    const bool on = g0 + g < grp;
    const seq_u32x4 r = seq_load16(A.q + n * A.q_n + head * A.q_h + 16 * c, on ? valid : 0, A.aln);
    sl[g] = on && A.slope ? A.slope[head] * kSeqLog2e : 0.f;
    m[g] = -INFINITY; l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) { q[g][i] = SeqElt<T>::get(r, i); acc[g][i] = 0.f; }
  }
  const char *kp = A.k + n * A.k_n + kvh * A.k_h + 16 * c, *vp = A.v + n * A.v_n + kvh * A.v_h + 16 * c;
  for (int k0 = beg; k0 < end; k0 += STEP) {
    seq_u32x4 kr[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = k0 + (u * NW + w) * KPW + kg;
      kr[u] = seq_load16(kp + key * A.k_t, key < end ? valid : 0, A.aln);
      vr[u] = seq_load16(vp + key * A.v_t, key < end ? valid : 0, A.aln);
    }
    float z[U][GT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = k0 + (u * NW + w) * KPW + kg;
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) s = fmaf(q[g][i], SeqElt<T>::get(kr[u], i), s);
#pragma unroll
        for (int o = 1; o < LPK; o <<= 1) s += __shfl_xor(s, o);
        s = A.cap > 0.f ? capl * tanhf(s * mul) : s * mul;
        if (A.slope) s = fmaf(-sl[g], (float)(len - 1 - key), s);
        z[u][g] = key < end ? s : -INFINITY;
      }
    }
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float mn = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, z[u][g]);
      const float ms = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m[g] - ms);
      m[g] = mn; l[g] *= al;
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[g][i] *= al;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = __builtin_amdgcn_exp2f(z[u][g] - ms);
        l[g] += p;
#pragma unroll
        for (int i = 0; i < EPL; ++i) acc[g][i] = fmaf(p, SeqElt<T>::get(vr[u], i), acc[g][i]);
      }
    }
  }
  // merge the lane groups of the wave, then the waves
#pragma unroll
  for (int g = 0; g < GT; ++g) {
#pragma unroll
    for (int o = LPK; o < 64; o <<= 1) {
      const float mo = __shfl_xor(m[g], o), lo = __shfl_xor(l[g], o), mn = fmaxf(m[g], mo), ms = mn == -INFINITY ? 0.f : mn;
      const float a = __builtin_amdgcn_exp2f(m[g] - ms), b = __builtin_amdgcn_exp2f(mo - ms);
      l[g] = l[g] * a + lo * b;
      m[g] = mn;
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
      if (c == 0) { stat[(w * GT + g) * 2] = m[g]; stat[(w * GT + g) * 2 + 1] = l[g]; }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < GT * LPK * EPL; i += 256) {
    const int g = i / (LPK * EPL), col = i % (LPK * EPL), head = kvh * grp + g0 + g;
    if (g0 + g >= grp || col >= A.d) continue;
    float mn = -INFINITY, ls = 0.f, o = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) mn = fmaxf(mn, stat[(x * GT + g) * 2]);
    const float ms = mn == -INFINITY ? 0.f : mn;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float f = __builtin_amdgcn_exp2f(stat[(x * GT + g) * 2] - ms);
      ls = fmaf(stat[(x * GT + g) * 2 + 1], f, ls);
      o = fmaf(sm[(x * GT + g) * LPK * EPL + col], f, o);
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

// rows of the cache that one workgroup takes: about 2048 workgroups at full length, 64 rows at least
int seq_step_chunk(int n, int hq, int hk, int capacity) {
  const int grp = hq / hk, gt = grp <= 1 ? 1 : grp <= 2 ? 2 : grp <= 4 ? 4 : 8;
  const int64_t per = (int64_t)n * hk * ((grp + gt - 1) / gt);
  const int64_t want = (per * capacity + 2047) / 2048;
  const int64_t chunk = (want + 63) / 64 * 64;
  return (int)(chunk < 64 ? 64 : chunk);
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
