// kernels_seq_misc.hip -- per-head norm + rotary positions of queries and keys, and dropout with the residual sum.
#include "kernels_seq.h"

namespace sttran {

// ---- rotary positions ------------------------------------------------------------------------------------------------------
// y = R(pos) x' with x' = w * x / sqrt(mean(x^2) + eps) (or x' = x without a norm).  R turns pair i of the first `rot` columns by
// pos * freq_i; the pair is (2i, 2i + 1) (interleaved) or (i, i + rot / 2) (halves); columns from rot on pass.
// Bound by memory: one read and one write of q and k.  A workgroup takes TT tokens at a time with all their heads, so an
// angle's cosine and sine are taken once a token: in 64 bits up to the turn's fraction (a far position times a frequency
// has no exact fraction in 32), then in fp32.  LPR lanes hold one row, 16 bytes each; a pair's other half comes through LDS.
template <int LPR>
struct SeqRot {
  static constexpr int kRows = 256 / LPR;                 // rows in flight
  int rot, half;
  bool inter;
  float* row;                                             // this row's LDS copy, rounded up to whole chunks
  // out[i] = the turned value of column e0 + i; sign -1: the turn back
  template <int EPL>
  __device__ __forceinline__ void turn(float (&x)[EPL], const float* cs, float sign, int c) const {
    const int e0 = c * EPL;
    if (inter) {
#pragma unroll
      for (int j = 0; j < EPL / 2; ++j) {
        const int i = e0 / 2 + j;
        if (i >= half) continue;
        const float co = cs[2 * i], si = sign * cs[2 * i + 1], a = x[2 * j], b = x[2 * j + 1];
        x[2 * j] = a * co - b * si;
        x[2 * j + 1] = b * co + a * si;
      }
      return;
    }
    // rows live in one wave: its own LDS writes are visible to it once they are done
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < EPL; ++j) row[e0 + j] = x[j];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = e0 + j;
      if (e >= rot) continue;
      const bool first = e < half;
      const int i = first ? e : e - half;
      const float other = row[first ? e + half : i], co = cs[2 * i], si = sign * cs[2 * i + 1];
      x[j] = first ? x[j] * co - other * si : x[j] * co + other * si;
    }
    __builtin_amdgcn_wave_barrier();
  }
};

__device__ __forceinline__ void seq_angles(const SeqRotaryArgs& A, float* cs, int64_t t0, int tt) {
  const int half = A.rot / 2;
  for (int i = threadIdx.x; i < tt * half; i += 256) {
    const int t = i / half, f = i % half;
    float co = 1.f, si = 0.f;
    if (t0 + t < A.tokens) {
      const double turns = (double)A.pos[t0 + t] * ((double)A.freq[f] * 0.15915494309189533577);   // 1 / (2 pi)
      const float frac = (float)(turns - rint(turns));
      sincospif(2.f * frac, &si, &co);
    }
    cs[2 * i] = co; cs[2 * i + 1] = si;
  }
}

template <class T, int LPR, bool BWD>
__global__ void __launch_bounds__(256) seq_rotary_kernel(SeqRotaryArgs A, int TT) {
  constexpr int EPL = SeqElt<T>::kPer16, ROWS = 256 / LPR;
  extern __shared__ __attribute__((aligned(16))) float sm[];
  float* cs = sm;                                          // [TT][rot / 2][2]
  const int rowlen = LPR * EPL, c = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
  SeqRot<LPR> R{A.rot, A.rot / 2, A.interleaved != 0, sm + (TT * A.rot + 3) / 4 * 4 + r0 * rowlen};
  const int heads = A.heads[0] + A.heads[1], dbytes = A.d * (int)sizeof(T), valid = dbytes - 16 * c;
  float dw[2][EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) dw[0][j] = dw[1][j] = 0.f;

  for (int64_t t0 = (int64_t)blockIdx.x * TT; t0 < A.tokens; t0 += (int64_t)gridDim.x * TT) {
    __syncthreads();
    seq_angles(A, cs, t0, TT);
    __syncthreads();
    const int rows = TT * heads;
    for (int b = 0; b < rows; b += ROWS) {
      const int r = b + r0, t = min(r, rows - 1) / heads, hh = min(r, rows - 1) % heads;
      const int which = hh >= A.heads[0] ? 1 : 0, head = which ? hh - A.heads[0] : hh;
      const int64_t token = t0 + t;
      const bool on = r < rows && token < A.tokens;
      const float* cst = cs + t * A.rot;
      const float* w = A.w[which];
      const int64_t at = (token * A.heads[which] + head) * dbytes + 16 * c;
      float x[EPL], inv = 1.f;
      const bool need_x = !BWD || w;
      seq_u32x4 xr = {0, 0, 0, 0};
      if (need_x) xr = seq_load16(A.x[which] + token * A.x_t[which] + head * A.x_h[which] + 16 * c, on ? valid : 0, A.aln);
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[j] = SeqElt<T>::get(xr, j);
      float wj[EPL];
      if (w) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          s = fmaf(x[j], x[j], s);
          wj[j] = c * EPL + j < A.d ? w[c * EPL + j] : 0.f;
        }
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) s += __shfl_xor(s, o);
        inv = 1.f / sqrtf(s / (float)A.d + A.eps);
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[j] *= inv;
      }
      float y[EPL];
      if constexpr (!BWD) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) y[j] = w ? x[j] * wj[j] : x[j];
        R.template turn<EPL>(y, cst, 1.f, c);
      } else {
        const seq_u32x4 gr = seq_load16(A.dy[which] + token * A.dy_t[which] + head * A.dy_h[which] + 16 * c, on ? valid : 0, A.aln);
        float g[EPL];
#pragma unroll
        for (int j = 0; j < EPL; ++j) g[j] = SeqElt<T>::get(gr, j);
        R.template turn<EPL>(g, cst, -1.f, c);
        if (w) {
          float s = 0.f;
#pragma unroll
          for (int j = 0; j < EPL; ++j) {
            const float gx = g[j] * x[j];
            if (which) dw[1][j] += gx; else dw[0][j] += gx;
            s = fmaf(gx, wj[j], s);
          }
#pragma unroll
          for (int o = 1; o < LPR; o <<= 1) s += __shfl_xor(s, o);
          s /= (float)A.d;
#pragma unroll
          for (int j = 0; j < EPL; ++j) y[j] = inv * (g[j] * wj[j] - x[j] * s);
        } else {
#pragma unroll
          for (int j = 0; j < EPL; ++j) y[j] = g[j];
        }
      }
      seq_u32x4 out = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < EPL; ++j) SeqElt<T>::put(out, j, y[j]);
      if (on) seq_store16((BWD ? A.dx[which] : A.y[which]) + at, out, valid, A.aln);
    }
  }
  if constexpr (BWD) {
    if (!A.part) return;
    // this workgroup's share of the weight gradients: rows in the order r0 = 0, 1, ...
    float* buf = sm;                                       // [ROWS][rowlen]
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < EPL; ++j) buf[r0 * rowlen + c * EPL + j] = dw[which][j];
      __syncthreads();
      for (int e = threadIdx.x; e < A.d; e += 256) {
        float s = 0.f;
        for (int r = 0; r < ROWS; ++r) s += buf[r * rowlen + e];
        A.part[((int64_t)blockIdx.x * 2 + which) * A.d + e] = s;
      }
    }
  }
}

// joins the workgroups' shares in a fixed order, in 64 bits: one workgroup 64 columns, four partial sums a column
__global__ void __launch_bounds__(256) seq_rotary_dw_kernel(SeqRotaryArgs A, int groups) {
  __shared__ double sm[256];
  const int which = blockIdx.y, e = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
  double s = 0.;
  if (e < A.d)
    for (int g = q; g < groups; g += 4) s += A.part[((int64_t)g * 2 + which) * A.d + e];
  sm[threadIdx.x] = s;
  __syncthreads();
  if (q == 0 && e < A.d && A.dw[which]) A.dw[which][e] = (float)(((sm[threadIdx.x] + sm[threadIdx.x + 64]) + sm[threadIdx.x + 128]) + sm[threadIdx.x + 192]);
}

static int rotary_tt(const SeqRotaryArgs& A) { return A.tokens >= 4096 ? 4 : 1; }
int seq_rotary_groups(const SeqRotaryArgs& A) {
  const int64_t tiles = (A.tokens + rotary_tt(A) - 1) / rotary_tt(A);
  return (int)(tiles < 1024 ? tiles : 1024);
}

template <class T, bool BWD>
static hipError_t rotary(hipStream_t s, const SeqRotaryArgs& A) {
  const int tt = rotary_tt(A), chunks = (A.d * (int)sizeof(T) + 15) / 16;
  const int64_t tiles = (A.tokens + tt - 1) / tt;
  const unsigned grid = BWD ? (unsigned)seq_rotary_groups(A) : (unsigned)(tiles < 16384 ? tiles : 16384);
  const int lds = ((tt * A.rot + 3) / 4 * 4 + 256 * SeqElt<T>::kPer16) * 4;        // angles + rows (or the gradient's shares)
  if (chunks <= 8) seq_rotary_kernel<T, 8, BWD><<<grid, 256, lds, s>>>(A, tt);
  else if (chunks <= 16) seq_rotary_kernel<T, 16, BWD><<<grid, 256, lds, s>>>(A, tt);
  else if (chunks <= 32) seq_rotary_kernel<T, 32, BWD><<<grid, 256, lds, s>>>(A, tt);
  else if constexpr (sizeof(T) == 4) seq_rotary_kernel<T, 64, BWD><<<grid, 256, lds, s>>>(A, tt);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !BWD || !A.part) return e;
  seq_rotary_dw_kernel<<<dim3((unsigned)((A.d + 63) / 64), 2), 256, 0, s>>>(A, (int)grid);
  return hipGetLastError();
}

hipError_t launch_seq_rotary_forward(hipStream_t s, int bf16, const SeqRotaryArgs& A) {
  if (A.tokens == 0) return hipSuccess;
  return bf16 ? rotary<__bf16, false>(s, A) : rotary<float, false>(s, A);
}
hipError_t launch_seq_rotary_backward(hipStream_t s, int bf16, const SeqRotaryArgs& A) {
  if (A.tokens == 0) {                                     // no rows: the weights' gradients are zeros all the same
    if (!A.part) return hipSuccess;
    seq_rotary_dw_kernel<<<dim3((unsigned)((A.d + 63) / 64), 2), 256, 0, s>>>(A, 0);
    return hipGetLastError();
  }
  return bf16 ? rotary<__bf16, true>(s, A) : rotary<float, true>(s, A);
}

// ---- dropout ---------------------------------------------------------------------------------------------------------------
// y_i = res_i + (word_i >= threshold ? x_i * mul : 0).  word_i comes from the counter-based generator Philox 4x32 with 10 rounds
// (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011): block i / 4 has the 128-bit counter
// (i / 4, offset) under the 64-bit key and gives the words of four elements, so the mask is a function of (key, offset, i) and
// is never stored.  Bound by memory: x and res in, y out; 10 rounds are 20 wide multiplies for four elements.
__device__ __forceinline__ void seq_philox(uint64_t block, uint64_t offset, uint64_t key, uint32_t (&out)[4]) {
  uint32_t x0 = (uint32_t)block, x1 = (uint32_t)(block >> 32), x2 = (uint32_t)offset, x3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)x0 * 0xD2511F53u, b = (uint64_t)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ k0; x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ k1; x3 = (uint32_t)a;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
  out[0] = x0; out[1] = x1; out[2] = x2; out[3] = x3;
}

template <class T>
__global__ void __launch_bounds__(256) seq_dropout_kernel(SeqDropoutArgs A) {
  constexpr int EPL = SeqElt<T>::kPer16;
  const int64_t key = A.rng ? A.rng[0] : A.key, offset = A.rng ? A.rng[1] : A.offset;
  const int64_t chunks = (A.n + EPL - 1) / EPL;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
    const int64_t left = (A.n - i * EPL) * (int64_t)sizeof(T);
    const int valid = left < 16 ? (int)left : 16;
    const seq_u32x4 x = seq_load16(A.x + i * 16, valid, A.aln);
    seq_u32x4 r = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    if (A.res) r = seq_load16(A.res + i * 16, valid, A.aln);
#pragma unroll
    for (int b = 0; b < EPL / 4; ++b) {
      uint32_t word[4];
      seq_philox((uint64_t)i * (EPL / 4) + b, (uint64_t)offset, (uint64_t)key, word);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = word[j] >= A.threshold ? SeqElt<T>::get(x, 4 * b + j) * A.mul : 0.f;
        SeqElt<T>::put(y, 4 * b + j, A.res ? SeqElt<T>::get(r, 4 * b + j) + v : v);
      }
    }
    seq_store16(A.y + i * 16, y, valid, A.aln);
  }
  if (A.used && blockIdx.x == 0 && threadIdx.x == 0) { A.used[0] = key; A.used[1] = offset; }
}

hipError_t launch_seq_dropout(hipStream_t s, int bf16, const SeqDropoutArgs& A) {
  const int64_t chunks = (A.n + (bf16 ? 7 : 3)) / (bf16 ? 8 : 4), blocks = (chunks + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 1 ? 1 : blocks < 16384 ? blocks : 16384);
  if (bf16) seq_dropout_kernel<__bf16><<<grid, 256, 0, s>>>(A);
  else seq_dropout_kernel<float><<<grid, 256, 0, s>>>(A);
  return hipGetLastError();
}

}  // namespace sttran
