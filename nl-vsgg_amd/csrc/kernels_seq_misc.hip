// kernels_seq_misc.hip -- per-head norm + rotary positions of queries and keys, and dropout with the residual sum.
#include "kernels_seq.h"

namespace sttran {

// ---- rotary positions ------------------------------------------------------------------------------------------------------
// y = R(pos) x' with x' = w * x / sqrt(mean(x^2) + eps) (or x' = x without a norm).  R turns pair i of the first `rot` columns by
// pos * freq_i; the pair is (2i, 2i + 1) (interleaved) or (i, i + rot / 2) (halves); columns from rot on pass:
//   y[e] = x'[e] * C[e] + x'[partner(e)] * S[e],   C = cos, S = -sin / +sin on a pair's first / second column, 1 and 0 behind rot.
// The backward pass turns dy back (S negated) and takes the norm's gradient from it.
// Bound by memory: one read and one write of q and k (and of their gradients).  A workgroup takes TT tokens at a time with all
// their heads, so C and S are made once a token: the angle in 64 bits up to the turn's fraction (a far position times a frequency
// has no exact fraction in 32), then in fp32.  LPR lanes hold one row, 16 bytes each; the halves' partners come through LDS.
// What bounds it is the bytes in flight, so registers are kept low for more waves: 8 a SIMD forward (110 us at 7), 5 backward (166 us
// at 4); the rows' next pass fetched ahead cost registers and was slower (135 / 266 us), and so were larger grids.
// Non-temporal stores: 249 -> 236 us for both passes by themselves, but the attention that reads the result next loses it (64 x 512 rows,
// the two together 301 -> 304 us): plain ones.
// Measured (32768 tokens, 16 + 4 heads of 128 columns, 96 turned, bfloat16, norm): 90 us forward (3.7 TB/s), 147 us backward (3.4 TB/s) and
// 7 us for the weights' gradients.
template <class T, int LPR, bool BWD>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(BWD ? 5 : 8, 8))) seq_rotary_kernel(SeqRotaryArgs A, int TT) {
  constexpr int EPL = SeqElt<T>::kPer16, ROWS = 256 / LPR, ROW = LPR * EPL;
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const int c = threadIdx.x % LPR, r0 = threadIdx.x / LPR, e0 = c * EPL, half = A.rot / 2;
  float* const wts = sm + TT * 2 * ROW;                    // behind the angles [TT][C | S][ROW]: the weights of q and of k,
  float* const row = wts + 2 * ROW + r0 * ROW;             // then a copy of this lane's row
  const int heads = A.heads[0] + A.heads[1], dbytes = A.d * (int)sizeof(T), valid = dbytes - 16 * c;
  const bool norm = A.w[0] != nullptr, swap = !A.interleaved && A.rot > 0, chunked = half % EPL == 0;
  float dw[2][EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) dw[0][j] = dw[1][j] = 0.f;
  if (norm)
    for (int i = threadIdx.x; i < 2 * ROW; i += 256) wts[i] = i % ROW < A.d ? A.w[i / ROW][i % ROW] : 0.f;
  const float per_d = 1.f / (float)A.d;
  for (int i = threadIdx.x; i < TT * (ROW - A.rot); i += 256) {              // the columns that pass
    const int t = i / (ROW - A.rot), e = A.rot + i % (ROW - A.rot);
    sm[t * 2 * ROW + e] = 1.f;
    sm[t * 2 * ROW + ROW + e] = 0.f;
  }

  const int rows = TT * heads;
  struct Where { int t, which, head; int64_t token; bool on; };
  const auto where = [&](int64_t t0, int b) __attribute__((always_inline)) {
    const int r = min(b + r0, rows - 1);
    Where p;
    p.t = heads > 1 ? (int)__umulhi((uint32_t)r, A.per_head) : r;
    const int hh = r - p.t * heads;
    p.which = hh >= A.heads[0] ? 1 : 0;
    p.head = p.which ? hh - A.heads[0] : hh;
    p.token = t0 + p.t < A.tokens ? t0 + p.t : A.tokens - 1;
    p.on = b + r0 < rows && t0 + p.t < A.tokens;
    return p;
  };
  for (int64_t t0 = (int64_t)blockIdx.x * TT; t0 < A.tokens; t0 += (int64_t)gridDim.x * TT) {
    __syncthreads();
    for (int i = threadIdx.x; i < TT * half; i += 256) {
      const int t = i / half, f = i % half;
      const int64_t token = t0 + t < A.tokens ? t0 + t : A.tokens - 1;
      const double turns = (double)A.pos[token] * ((double)A.freq[f] * 0.15915494309189533577);   // 1 / (2 pi)
      float co, si;
      sincospif(2.f * (float)(turns - rint(turns)), &si, &co);
      float* C = sm + t * 2 * ROW;
      const int a = A.interleaved ? 2 * f : f, b = A.interleaved ? a + 1 : f + half;
      C[a] = co; C[b] = co;
      C[ROW + a] = BWD ? si : -si; C[ROW + b] = BWD ? -si : si;
    }
    __syncthreads();
    for (int b = 0; b < rows; b += ROWS) {
      const Where p = where(t0, b);
      seq_u32x4 xr = {0, 0, 0, 0}, gr = {0, 0, 0, 0};
      if (!BWD || norm) xr = seq_row_chunk(A.x[p.which] + p.token * A.x_t[p.which] + p.head * A.x_h[p.which], c, dbytes, A.aln);
      if (BWD) gr = seq_row_chunk(A.dy[p.which] + p.token * A.dy_t[p.which] + p.head * A.dy_h[p.which], c, dbytes, A.aln);
      const int t = p.t, which = p.which;
      const bool on = p.on;
      const int64_t at = (p.token * A.heads[which] + p.head) * dbytes;
      float x[EPL], y[EPL], wj[EPL], inv = 1.f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        x[j] = SeqElt<T>::get(xr, j);
        wj[j] = 1.f;
      }
      if (norm) {
#pragma unroll
        for (int j = 0; j < EPL; j += 4) {
          const seq_f32x4 a = *reinterpret_cast<const seq_f32x4*>(wts + which * ROW + e0 + j);
#pragma unroll
          for (int u = 0; u < 4; ++u) wj[j + u] = a[u];
        }
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) s = fmaf(x[j], x[j], s);
        inv = rsqrtf(seq_group_sum<LPR>(s) * per_d + A.eps);
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[j] *= inv;
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) y[j] = BWD ? SeqElt<T>::get(gr, j) : x[j] * wj[j];
      // the turn
      const float* C = sm + t * 2 * ROW + e0;
      float co[EPL], si[EPL], z[EPL];
#pragma unroll
      for (int j = 0; j < EPL; j += 4) {
        const seq_f32x4 a = *reinterpret_cast<const seq_f32x4*>(C + j), b4 = *reinterpret_cast<const seq_f32x4*>(C + ROW + j);
#pragma unroll
        for (int u = 0; u < 4; ++u) { co[j + u] = a[u]; si[j + u] = b4[u]; }
      }
      if (swap) {
        // a row lives in one wave, whose LDS accesses keep their order: only the compiler must
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < EPL; j += 4) *reinterpret_cast<seq_f32x4*>(row + e0 + j) = seq_f32x4{y[j], y[j + 1], y[j + 2], y[j + 3]};
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (chunked) {
          const float* p = row + (e0 < half ? e0 + half : e0 < A.rot ? e0 - half : e0);
#pragma unroll
          for (int j = 0; j < EPL; j += 4) {
            const seq_f32x4 a = *reinterpret_cast<const seq_f32x4*>(p + j);
#pragma unroll
            for (int u = 0; u < 4; ++u) z[j + u] = a[u];
          }
        } else {
#pragma unroll
          for (int j = 0; j < EPL; ++j) {
            const int e = e0 + j;
            z[j] = row[e < half ? e + half : e < A.rot ? e - half : e];
          }
        }
        __builtin_amdgcn_wave_barrier();
      } else {
#pragma unroll
        for (int j = 0; j < EPL; ++j) z[j] = y[j ^ 1];
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) z[j] = e0 + j < A.rot ? z[j] : 0.f;             // what passes has no partner, infinities neither
      seq_u32x4 out = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < EPL; ++j) y[j] = fmaf(z[j], si[j], y[j] * co[j]);
      if (BWD && norm) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const float gx = on ? y[j] * x[j] : 0.f;
          dw[0][j] += which ? 0.f : gx;
          dw[1][j] += which ? gx : 0.f;
          s = fmaf(y[j] * x[j], wj[j], s);
        }
        s = seq_group_sum<LPR>(s) * per_d;
#pragma unroll
        for (int j = 0; j < EPL; ++j) y[j] = inv * (y[j] * wj[j] - x[j] * s);
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) SeqElt<T>::put(out, j, y[j]);
      if (on) seq_store16((BWD ? A.dx[which] : A.y[which]) + at + 16 * c, out, valid, A.aln);
    }
  }
  if constexpr (BWD) {
    if (!A.part) return;
    // this workgroup's share of the weight gradients: rows in the order r0 = 0, 1, ...
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < EPL; ++j) sm[r0 * ROW + e0 + j] = dw[which][j];
      __syncthreads();
      for (int e = threadIdx.x; e < A.d; e += 256) {
        float s = 0.f;
        for (int r = 0; r < ROWS; ++r) s += sm[r * ROW + e];
        A.part[((int64_t)blockIdx.x * 2 + which) * A.d + e] = s;
      }
    }
  }
}

// joins the workgroups' shares in a fixed order, in 64 bits: one workgroup 64 columns, sixteen partial sums a column
__global__ void __launch_bounds__(1024) seq_rotary_dw_kernel(SeqRotaryArgs A, int groups) {
  __shared__ double sm[1024];
  const int which = blockIdx.y, e = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
  double s = 0.;
  if (e < A.d) {
    const float* p = A.part + (int64_t)which * A.d + e;
#pragma unroll 8
    for (int g = q; g < groups; g += 16) s += p[(int64_t)g * 2 * A.d];
  }
  sm[threadIdx.x] = s;
  __syncthreads();
  if (q == 0 && e < A.d && A.dw[which]) {
    for (int i = 1; i < 16; ++i) s += sm[threadIdx.x + 64 * i];
    A.dw[which][e] = (float)s;
  }
}

static int rotary_tt(const SeqRotaryArgs& A) { return A.tokens >= 4096 ? 4 : 1; }
int seq_rotary_groups(const SeqRotaryArgs& A) {
  const int64_t tiles = (A.tokens + rotary_tt(A) - 1) / rotary_tt(A);
  return (int)(tiles < 1280 ? tiles : 1280);
}

template <class T, int LPR, bool BWD>
static hipError_t rotary_lpr(hipStream_t s, SeqRotaryArgs A) {
  const int tt = rotary_tt(A), heads = A.heads[0] + A.heads[1];
  A.per_head = heads > 1 ? (uint32_t)(((uint64_t)1 << 32) / heads + 1) : 0;      // r / heads = high half of r * per_head
  const int64_t tiles = (A.tokens + tt - 1) / tt;
  const unsigned grid = BWD ? (unsigned)seq_rotary_groups(A) : (unsigned)(tiles < 2048 ? tiles : 2048);
  constexpr int row = LPR * SeqElt<T>::kPer16;
  const int lds = (tt * 2 * row + 2 * row + 256 / LPR * row) * 4;                // angles, weights, rows (or the gradient's shares)
  seq_rotary_kernel<T, LPR, BWD><<<grid, 256, lds, s>>>(A, tt);
  return hipGetLastError();
}
static hipError_t rotary_dw(hipStream_t s, const SeqRotaryArgs& A, int groups) {
  seq_rotary_dw_kernel<<<dim3((unsigned)((A.d + 63) / 64), 2), 1024, 0, s>>>(A, groups);
  return hipGetLastError();
}
template <class T, bool BWD>
static hipError_t rotary(hipStream_t s, const SeqRotaryArgs& A) {
  const int chunks = (A.d * (int)sizeof(T) + 15) / 16;
  hipError_t e = hipSuccess;
  if (chunks <= 8) e = rotary_lpr<T, 8, BWD>(s, A);
  else if (chunks <= 16) e = rotary_lpr<T, 16, BWD>(s, A);
  else if (chunks <= 32) e = rotary_lpr<T, 32, BWD>(s, A);
  else if constexpr (sizeof(T) == 4) e = rotary_lpr<T, 64, BWD>(s, A);
  return e != hipSuccess || !BWD || !A.part ? e : rotary_dw(s, A, seq_rotary_groups(A));
}

hipError_t launch_seq_rotary_forward(hipStream_t s, int bf16, const SeqRotaryArgs& A) {
  if (A.tokens == 0) return hipSuccess;
  return bf16 ? rotary<__bf16, false>(s, A) : rotary<float, false>(s, A);
}
hipError_t launch_seq_rotary_backward(hipStream_t s, int bf16, const SeqRotaryArgs& A) {
  if (A.tokens == 0) {                                     // no rows: the weights' gradients are zeros all the same
    return A.part ? rotary_dw(s, A, 0) : hipSuccess;
  }
  return bf16 ? rotary<__bf16, true>(s, A) : rotary<float, true>(s, A);
}

// ---- dropout ---------------------------------------------------------------------------------------------------------------
// y_i = res_i + (word_i >= threshold ? x_i * mul : 0).  word_i comes from the counter-based generator Philox 4x32 with 10 rounds
// (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011): block i / 4 has the 128-bit counter
// (i / 4, offset) under the 64-bit key and gives the words of four elements, so the mask is a function of (key, offset, i) and
// is never stored.  Bound by memory: x and res in, y out; 10 rounds are 20 wide multiplies for four elements.
// Measured (22528 x 4096, bfloat16, residual): 104 us forward, 5.3 TB/s, 68 us backward, 5.4: a large copy's rate.
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
    const int aln = valid & 3 ? 2 : A.aln;              // an odd number of 2-byte elements ends within a dword that is not all its own
    const seq_u32x4 x = seq_load16(A.x + i * 16, valid, aln);
    seq_u32x4 r = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    if (A.res) r = seq_load16(A.res + i * 16, valid, aln);
#pragma unroll
    for (int b = 0; b < EPL / 4; ++b) {
      uint32_t word[4];
      seq_philox((uint64_t)i * (EPL / 4) + b, (uint64_t)offset, (uint64_t)key, word);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = word[j] >= A.threshold && !A.none ? SeqElt<T>::get(x, 4 * b + j) * A.mul : 0.f;
        SeqElt<T>::put(y, 4 * b + j, A.res ? SeqElt<T>::get(r, 4 * b + j) + v : v);
      }
    }
    seq_store16(A.y + i * 16, y, valid, aln);
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
