// kernels_seq_attn.hip -- attention over packed sequences, forward.
//   o_i = sum_j p_ij v_j,  p_i = softmax over the visible keys j of z_ij,
//   z_ij = cap * tanh(scale * q_i.k_j / cap) - slope_h * |place_i - j|
#include "kernels_seq.h"
#include "seq_attn.h"

namespace sttran {

// the own rows in `rows`, key by key over what each of them sees in [beg, end)
template <class C>
__device__ __forceinline__ void seq_attn_fwd_again(const SeqAttnArgs& A, const SeqScore& sc, uint32_t rows, SeqRow me, int row0, int head,
                                                             int beg, int end, int dh) {
  using T = typename C::E;
  const int lane = threadIdx.x & 63, kvh = head / (A.hq / A.hk);
#pragma unroll 1
  for (int n = 0; n < 32; ++n) {
    const int row = row0 + n;
    if (!(rows >> n & 1) || row >= A.tq || n % C::DS != dh) continue;
    const int lo = max(__shfl(me.lo, n), beg), hi = min(__shfl(me.hi, n), end), base = __shfl(me.base, n);
    const SeqSpread q = seq_spread<T>(A.raw[0].p + head * A.raw[0].h + (int64_t)row * A.raw[0].t, A.d);
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f}, unused;
#pragma unroll 1
    for (int key = lo; key < hi; ++key) {
      const SeqSpread k = seq_spread<T>(A.raw[1].p + kvh * A.raw[1].h + (int64_t)key * A.raw[1].t, A.d);
      const SeqSpread v = seq_spread<T>(A.raw[2].p + kvh * A.raw[2].h + (int64_t)key * A.raw[2].t, A.d);
      const float z = seq_z(A, sc, seq_spread_dot(q, k), base, key, unused);
      const float mn = fmaxf(m, z), ms = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - ms), p = __builtin_amdgcn_exp2f(z - ms);
      l = fmaf(l, al, p);
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = fmaf(o[u], al, p * v.x[u]);
      m = mn;
      if (!(l == l)) break;                          // a NaN probability: all of the row is NaN, whatever follows
    }
    if (A.splits > 1) {
      const int64_t at = ((int64_t)blockIdx.y * A.hq + head) * A.tq + row;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (lane + 64 * u < A.d) A.part[at * A.d + lane + 64 * u] = o[u];
      float* ps = A.part + (int64_t)A.splits * A.hq * A.tq * A.d + at * 2;
      if (lane == 0) { ps[0] = m; ps[1] = l; }
      continue;
    }
    const int64_t at = ((int64_t)row * A.hq + head) * A.d * C::OS;
    seq_spread_store<T>(A.out + at, A.out_lo ? A.out_lo + at : nullptr, o, l == 0.f ? 0.f : 1.f / l, A.d);
    if (A.lse && lane == 0) A.lse[(int64_t)head * A.tq + row] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
  }
}

// One pass over the keys with the running maximum m and sum l of the softmax (both fp32, base 2).  The accumulator is rescaled
// only when the maximum grows by more than 8 (a factor of 256): p stays below 2^8 and the final division by l undoes any
// common factor exactly as the textbook form does.
// N scores of one row, x[i] of key k0 + 8 (i / 4) + i % 4, become what z is linear in -- z = c1 * x + c0 -- so that one fma stands
// before the exponential; hidden ones become -inf (c1 > 0); returns the largest z.  SLOPE: distances, or a scale that is not positive.
//   neither: the products;  kSeqCapNear alone: -1 / (1 + e^(2 products)), z = cap - 2 cap / (1 + ..);  else: z itself
template <class C, int CAP, bool SLOPE, int N>
__device__ __forceinline__ float seq_bend(const SeqAttnArgs& A, const SeqScore& sc, float (&x)[N], int k0, int base, bool full, int lo, int hi,
                                          float& c1, float& c0) {
  if constexpr (CAP == kSeqCapNone && !SLOPE) {
    c1 = sc.mul; c0 = 0.f;
  } else if constexpr (CAP == kSeqCapNear && !SLOPE) {
    c1 = 2.f * sc.capl; c0 = sc.capl;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = -__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x[i] * (sc.mul * (2.f * kSeqLog2e))));
  } else {
    c1 = 1.f; c0 = 0.f;
    if constexpr (CAP != kSeqCapNone) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = sc.capl * seq_tanh<CAP == kSeqCapNear>(x[i] * sc.mul);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] *= sc.mul;
    }
    if constexpr (SLOPE) {
      const float at = (float)(base - k0);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = fmaf(-sc.slope, fabsf(at - (float)(8 * (i >> 2) + (i & 3))), x[i]);
    }
  }
  if (!full) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int key = k0 + 8 * (i >> 2) + (i & 3);
      x[i] = key >= lo && key < hi ? x[i] : -INFINITY;
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
  return fmaf(m, c1, c0);
}

template <class C>
struct SeqFwdLds {                                       // DS == 1: two tiles of keys and of values; else one of each and the exchange
  static constexpr int kBufs = C::DS == 1 ? 2 : 1;
  // the workgroup's small notes before and after the loop lie where the exchange is during it: at DP = 256 in fp32 two workgroups
  // then share a CU's 160 KB
  static constexpr int kXch = 2 * kBufs * C::kTileBytes, kRed = kXch, kRefs = kXch + (C::DS > 1 ? C::NW * SeqShare<C, 1>::kWave : 0);
  static constexpr int kBytes = C::DS > 1 ? kRefs + C::NW * 128 : kXch + C::NW * 8;
};
// Bound by the matrix pipe where sequences are long -- two products of 2 d operations a visible pair, 4 bytes of LDS read for every 32
// operations, scores and probabilities never leave the registers -- and by the latency of a workgroup's few blocks where they are short.
// Measured (a large matrix product reaches 1182 TFLOP/s in bfloat16 and 154 in fp32 on the card):
//   three sequences of 4000 .. 8000 rows, 8 heads over 2 of 128 columns, causal, bfloat16: 305 us, 870 TFLOP/s;
//   capped, 16 heads over 4: 680 us, 730 TFLOP/s (the exponential and the reciprocal of each score's tanh: vector units busy 0.59 of the
//   time, where it is 0.40 without a cap; 730 us at the clocks of a profiled run);  a cap above 1024: 663 us where 50 takes 380
//   96 of 37 .. 500 rows, 8 over 2 of 64, distances: 66 us (vector units 0.46, matrix pipe 0.11)
//   four of 1800 .. 2240 rows, 8 heads of 242, distances, fp32 on planes: 1150 us (six products for one)
//   1024 of 5 .. 35, 8 of 242, fp32 instructions: 255 us, 2.5 TB/s
// 32 own rows a wave: the stationary operand stays in registers, so every value read from LDS serves 32 rows.
template <class C, int CAP, bool SLOPE, bool TWO>
__global__ void __launch_bounds__(C::NT) __attribute__((amdgpu_waves_per_eu(2, 2)))
seq_attn_fwd_kernel(SeqAttnArgs A) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* xch = smem + SeqFwdLds<C>::kXch;
  int* red = reinterpret_cast<int*>(smem + SeqFwdLds<C>::kRed);
  float* refs = reinterpret_cast<float*>(smem + SeqFwdLds<C>::kRefs);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int tiles = (A.tq + C::RB - 1) / C::RB;
  const int id = seq_xcd_order(blockIdx.x, gridDim.x);
  // rows that see most keys first where the order masks
  const int head = id / tiles, tile = tiles - 1 - seq_spread_tile(A, id % tiles, tiles, A.hq);
  const int kvh = head / (A.hq / A.hk), dh = w % C::DS;
  const int row0 = tile * C::RB + 32 * (w / C::DS), row = row0 + (lane & 31);
  const int dbytes = C::row_bytes(A.d);

  const SeqRow me = seq_row_of_wave(A, row0, row);
  int lo = me.hi > me.lo ? me.lo : INT_MAX, hi = me.hi;
  seq_wave_range(lo, hi);
  const int wlo = lo, whi = hi;                                     // what this wave's rows see
  if (lane == 0) { red[2 * w] = lo; red[2 * w + 1] = hi; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < C::NW; ++i) { lo = min(lo, red[2 * i]); hi = max(hi, red[2 * i + 1]); }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  int beg = lo, end = max(hi, lo);
  if (hi <= 0) beg = end = 0;
  if (A.splits > 1) {                                               // this workgroup's share of the keys, whole tiles
    const int per = ((end - beg + A.splits - 1) / A.splits + C::BR - 1) / C::BR * C::BR;
    beg = min(beg + (int)blockIdx.y * per, end);
    end = min(beg + per, end);
  }

  const char *kp = A.k + kvh * A.k_h, *vp = A.v + kvh * A.v_h;
  SeqMover mk, mv;
  mk.init<C>(A.k_t, dbytes);
  mv.init<C>(A.v_t, dbytes);
  char *kt_lds = smem, *vt_lds = smem + C::kTileBytes;
  if (beg < end) {
    seq_tile_move<C>(mk, kt_lds, kp, A.k_t, beg, end, dbytes);
    seq_tile_move<C>(mv, vt_lds, vp, A.v_t, beg, end, dbytes);
  }
  seq_u32x4 own[C::PL * C::NF];
  seq_own_load<C>(own, A.q + head * A.q_h, A.q_t, row0, A.tq, dh, dbytes);
  const SeqScore sc(A, head);
  const int rlo = max(me.lo, beg), rhi = min(me.hi, end);           // this lane's visible keys of this workgroup
  seq_f32x16 acc[C::NB];
#pragma unroll
  for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[nb][e] = 0.f;
  float m = -INFINITY, l = 0.f;
  seq_tile_done<C>(mk, kt_lds, dbytes);
  seq_tile_done<C>(mv, vt_lds, dbytes);
  __syncthreads();

  for (int kt = beg, buf = 0; kt < end; kt += C::BR) {
    const bool more = kt + C::BR < end, active = wlo < min(kt + C::BR, end) && whi > kt;
    char *kn = kt_lds, *vn = vt_lds;
    if constexpr (C::DS == 1) {
      kn = smem + (buf ^ 1) * 2 * C::kTileBytes;
      vn = kn + C::kTileBytes;
      if (more) {
        seq_tile_move<C>(mk, kn, kp, A.k_t, kt + C::BR, end, dbytes);
        seq_tile_move<C>(mv, vn, vp, A.v_t, kt + C::BR, end, dbytes);
      }
    }
    seq_f32x16 s[C::NSUB];
    if (active) {
#pragma unroll
      for (int u = 0; u < C::NSUB; ++u) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[u][e] = 0.f;
        seq_scores<C>(s[u], kt_lds, u, dh, own);
      }
    }
    const bool full = __all(rlo <= kt && rhi >= kt + C::BR);
    float c1, c0;
    if constexpr (C::DS == 1) {
      if (active) {
        float x[16 * C::NSUB];
#pragma unroll
        for (int i = 0; i < 16 * C::NSUB; ++i) x[i] = s[i >> 4][i & 15];
        float mt = seq_bend<C, CAP, SLOPE>(A, sc, x, kt + 4 * h, me.base, full, rlo, rhi, c1, c0);
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        if (__any(mt > m + 8.f || (m == -INFINITY && mt > -INFINITY))) {
          const float mn = fmaxf(m, mt);
          const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
          m = mn; l *= al;
#pragma unroll
          for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[nb][e] *= al;
        }
        c0 -= m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < C::NSUB; ++u) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[u][e] = __builtin_amdgcn_exp2f(fmaf(x[16 * u + e], c1, c0));
            l += s[u][e];
          }
          seq_reduce<C, TWO>(acc, vt_lds, u, dh, s[u]);
        }
      }
    } else {
      // Each wave of the team adds up and exponentiates its share of the block's quads, against the team's maximum so far, or its own
      // where that is 2^30 behind; it tells the others which.  So one barrier brings probabilities, and the rare change of the
      // maximum is made afterwards by factors.
      static_assert(C::NSUB == 1, "one block is exchanged");
      using S = SeqShare<C, 1>;
      const int first = w - dh;
      if (active) S::put(s[0], xch, first, dh, 0);
      seq_tile_done<C>(mv, vt_lds, dbytes);
      __syncthreads();                                               // keys are free, values and partial scores are there
      if (more) seq_tile_move<C>(mk, kn, kp, A.k_t, kt + C::BR, end, dbytes);
      float part = 0.f;
      if (active) {
        float x[4 * S::GP];
#pragma unroll
        for (int i = 0; i < S::GP; ++i) {
          const seq_f32x4 q = S::sum(s[0], xch, first, dh, 0, i);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * i + e] = q[e];
        }
        float mt = seq_bend<C, CAP, SLOPE>(A, sc, x, kt + 8 * dh * S::GP + 4 * h, me.base, full, rlo, rhi, c1, c0);
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const float ref = mt > m + 30.f ? mt : m;
        c0 -= ref == -INFINITY ? 0.f : ref;
#pragma unroll
        for (int i = 0; i < S::GP; ++i) {
          seq_f32x4 p;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(x[4 * i + e], c1, c0));
            part += p[e];
          }
          S::leave(p, xch, first, dh, 0, i);
        }
        if (h == 0) refs[w * 32 + lane] = ref;
      }
      __syncthreads();
      if (active) {
        float r[C::DS], mn = -INFINITY, own = 0.f;
#pragma unroll
        for (int j = 0; j < C::DS; ++j) {
          r[j] = refs[(first + j) * 32 + (lane & 31)];
          mn = fmaxf(mn, r[j]);
          own = j == dh ? r[j] : own;
        }
        bool same = mn == m;
#pragma unroll
        for (int j = 0; j < C::DS; ++j) same = same && r[j] == mn;
        S::take(s[0], xch, first, 0);
        if (!__all(same)) {
          const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
          l *= al;
#pragma unroll
          for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[nb][e] *= al;
          m = mn;
#pragma unroll
          for (int j = 0; j < C::DS; ++j) {
            const float f = r[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r[j] - mn);
#pragma unroll
            for (int e = 4 * j * S::GP; e < 4 * (j + 1) * S::GP; ++e) s[0][e] *= f;
          }
          part *= own == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own - mn);
        }
        l += part;
        seq_reduce<C, TWO>(acc, vt_lds, 0, dh, s[0]);
      }
    }
    if (more) {
      seq_tile_done<C>(mk, kn, dbytes);
      if constexpr (C::DS == 1) seq_tile_done<C>(mv, vn, dbytes);
    }
    __syncthreads();
    if constexpr (C::DS == 1) {
      buf ^= 1;
      kt_lds = kn; vt_lds = vn;
    } else {
      if (more) seq_tile_move<C>(mv, vt_lds, vp, A.v_t, kt + C::BR, end, dbytes);
    }
  }
  l += __shfl_xor(l, 32);
  if constexpr (C::DS > 1) {                           // the team's shares of the sum
    if (h == 0) refs[w * 32 + lane] = l;
    __syncthreads();
    l = refs[(w - dh) * 32 + (lane & 31)];
#pragma unroll
    for (int j = 1; j < C::DS; ++j) l += refs[(w - dh + j) * 32 + (lane & 31)];
  }
  const uint32_t bad = seq_bad_rows<C>(acc, 0, red);
  if (bad) seq_attn_fwd_again<C>(A, sc, bad, me, row0, head, beg, end, dh);
  if (row >= A.tq || (bad >> (lane & 31) & 1)) return;
  if (A.splits > 1) {
    // unnormalised share of this split: [split][head][row][d], then [split][head][row][2]
    const int64_t at = ((int64_t)blockIdx.y * A.hq + head) * A.tq + row;
    float* po = A.part + at * A.d;
#pragma unroll
    for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = dh * C::DH + 32 * nb + 8 * (e >> 2) + 4 * h + (e & 3);
        if (col < A.d) po[col] = acc[nb][e];
      }
    if (dh == 0 && h == 0) {
      float* ps = A.part + (int64_t)A.splits * A.hq * A.tq * A.d + at * 2;
      ps[0] = m; ps[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = ((int64_t)row * A.hq + head) * A.d * C::OS;
  seq_store_own<C>(acc, inv, A.out + at, A.out_lo ? A.out_lo + at : nullptr, dh, A.d, A.aln);
  if (A.lse && dh == 0 && h == 0) A.lse[(int64_t)head * A.tq + row] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// joins the shares of a launch that was split over the keys: one workgroup a (row, head).  The waves take the shares in turn, their
// sums are added in the order of the waves
template <class T>
__global__ void __launch_bounds__(256) seq_attn_join_kernel(SeqAttnArgs A, const int* lens, int chunk, int capacity) {
  __shared__ float sm[4][256], wt[256], red[8];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t i = blockIdx.x;                                            // head * tq + row
  const int head = (int)(i / A.tq), row = (int)(i % A.tq);
  const int64_t step = (int64_t)A.hq * A.tq;
  const int shares = lens ? min((min(max(lens[row], 1), capacity) + chunk - 1) / chunk, A.splits) : A.splits;
  const float *ps = A.part + (int64_t)A.splits * step * A.d + i * 2, *po = A.part + i * A.d;
  float m = -INFINITY;
  for (int s = tid; s < shares; s += 256) m = fmaxf(m, ps[s * step * 2]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) red[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ms = m == -INFINITY ? 0.f : m;
  float o[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
  for (int s0 = 0; s0 < shares; s0 += 256) {                               // a share that saw nothing weighs exp(-inf) = 0
    float f = 0.f;
    if (s0 + tid < shares) {
      f = __builtin_amdgcn_exp2f(ps[(s0 + tid) * step * 2] - ms);
      l = fmaf(ps[(s0 + tid) * step * 2 + 1], f, l);
    }
    __syncthreads();
    wt[tid] = f;
    __syncthreads();
    const int n = min(shares - s0, 256);
#pragma unroll 8
    for (int s = w; s < n; s += 4) {
      const float* p = po + (s0 + s) * step * A.d;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = fmaf(lane + 64 * u < A.d ? p[lane + 64 * u] : 0.f, wt[s], o[u]);
    }
  }
  l = seq_group_sum<64>(l);
  if (lane == 0) red[4 + w] = l;
#pragma unroll
  for (int u = 0; u < 4; ++u) sm[w][lane + 64 * u] = o[u];
  __syncthreads();
  l = ((red[4] + red[5]) + red[6]) + red[7];
  const int col = threadIdx.x;
  if (col < A.d) {
    const float x = (((sm[0][col] + sm[1][col]) + sm[2][col]) + sm[3][col]) * (l == 0.f ? 0.f : 1.f / l);
    const int64_t at = ((int64_t)row * A.hq + head) * A.d + col;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float*>(A.out)[at] = x;
    } else {
      const float y = SeqElt<T>::round(x);
      reinterpret_cast<uint16_t*>(A.out)[at] = (uint16_t)SeqElt<T>::bits(y);
      if (A.out_lo) reinterpret_cast<uint16_t*>(A.out_lo)[at] = (uint16_t)SeqElt<T>::bits(x - y);
    }
  }
  if (A.lse && threadIdx.x == 0) A.lse[i] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

hipError_t launch_seq_attn_join(hipStream_t s, int bf16, const SeqAttnArgs& A, const int* lens, int chunk, int capacity) {
  const unsigned grid = (unsigned)((int64_t)A.hq * A.tq);
  if (bf16) seq_attn_join_kernel<__bf16><<<grid, 256, 0, s>>>(A, lens, chunk, capacity);
  else seq_attn_join_kernel<float><<<grid, 256, 0, s>>>(A, lens, chunk, capacity);
  return hipGetLastError();
}

template <class C, int CAP, bool SLOPE, bool TWO>
static hipError_t fwd_as(hipStream_t s, const SeqAttnArgs& A) {
  constexpr int lds = SeqFwdLds<C>::kBytes;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  static DeviceMarks marks;
  auto fn = seq_attn_fwd_kernel<C, CAP, SLOPE, TWO>;
  hipError_t e = marks.raise_lds(reinterpret_cast<const void*>(fn), lds);
  if (e != hipSuccess) return e;
  const int tiles = (A.tq + C::RB - 1) / C::RB;
  fn<<<dim3((unsigned)(tiles * A.hq), (unsigned)A.splits), C::NT, lds, s>>>(A);
  e = hipGetLastError();
  return e != hipSuccess || A.splits == 1 ? e : launch_seq_attn_join(s, C::OS == 2, A, nullptr, 0, 0);
}

// A kernel for each of no cap and cap, no distances and distances: with the others' bodies beside its own in one kernel the registers
// spill and drain the loads in flight (three sequences of 4000 .. 8000 rows, 128 columns: forward 335 -> 307 us).  bfloat16 under a large
// cap, which bends hardly a score, has one: with distances, whose factor may be zero, and probabilities of 16 bits
template <class C, bool TWO = false>
static hipError_t fwd(hipStream_t s, const SeqAttnArgs& A) {
  const bool slope = A.slope || A.scale <= 0.f;          // without distances their factor is zero
  if constexpr (C::OS == 2) {
    if (A.cap > kSeqNearCap) return fwd_as<C, kSeqCap, true, true>(s, A);
  }
  constexpr int cap = C::OS == 2 ? kSeqCapNear : kSeqCap;
  if (A.cap > 0.f) return slope ? fwd_as<C, cap, true, TWO>(s, A) : fwd_as<C, cap, false, TWO>(s, A);
  return slope ? fwd_as<C, kSeqCapNone, true, TWO>(s, A) : fwd_as<C, kSeqCapNone, false, TWO>(s, A);
}

// Own rows a workgroup: 128 or (heads of 64 columns, whose calls have small tiles to spare: 84 -> 74 us on 96 sequences of 37 .. 500
// rows, 263 -> 254 us on three of 4000 .. 8000) 64 where a wave holds whole heads; 32 or 64 where teams of waves share them
template <class T, bool VEC, bool TWO>
static hipError_t pick(hipStream_t s, const SeqAttnArgs& A) {
  if (A.d <= 64) return fwd<SeqTile<T, 64, 1, 2, 64, VEC>, TWO>(s, A);
  if (A.d <= 128) return fwd<SeqTile<T, 128, 1, 4, sizeof(T) == 2 ? 64 : 32, VEC>, TWO>(s, A);
  return fwd<SeqTile<T, 256, sizeof(T) == 2 ? 2 : 4, 4, 32, VEC>, TWO>(s, A);
}
static hipError_t pick_planes(hipStream_t s, const SeqAttnArgs& A) {
  if (A.d <= 64) return fwd<SeqTile<float, 64, 1, 4, 32, true, 3>>(s, A);
  if (A.d <= 128) return fwd<SeqTile<float, 128, 2, 4, 32, true, 3>>(s, A);
  return fwd<SeqTile<float, 256, 4, 8, 32, true, 3>>(s, A);
}
int seq_attn_fwd_tile(int bf16, bool planes, int d) {
  if (planes) return d <= 64 ? 128 : 64;
  return d <= 64 ? 64 : d <= 128 ? 128 : bf16 ? 64 : 32;
}

// bfloat16 in sequences of fewer than 64 rows on average: probabilities enter the product with 16 bits (TWO; with 8 the result is 1.2 .. 1.4
// times as far off as its own rounding, with few rows up to 1.48, and dq, dk up to 1.73 through delta).  It costs a third of the products,
// which such calls hardly wait for (1000 x 32 rows, 8 heads of 64 columns, 43 -> 44 us; 500 x 60, 16 over 4 of 128, 136 -> 145; but three of
// 4000 .. 8000 rows 305 -> 396).  Rows at odd 2 bytes take 16 bits always.  The host knows the average alone: short sequences beside a
// long one get 8 bits too (ten of 5 .. 50 rows beside one of 8000: 1.1 .. 1.2 times their own rounding, their gradients 1.2 .. 1.5)
hipError_t launch_seq_attn_fwd(hipStream_t s, int bf16, bool planes, const SeqAttnArgs& A) {
  const bool vec = A.aln >= 4;
  if (planes) return pick_planes(s, A);
  if (bf16) return !vec ? pick<__bf16, false, true>(s, A) : seq_fewer_rows(A, 64) ? pick<__bf16, true, true>(s, A) : pick<__bf16, true, false>(s, A);
  return pick<float, true, false>(s, A);                // 4-byte elements are 4-byte aligned
}

}  // namespace sttran
