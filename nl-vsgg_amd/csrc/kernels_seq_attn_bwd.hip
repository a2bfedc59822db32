// kernels_seq_attn_bwd.hip -- gradients of attention over packed sequences (kernels_seq_attn.hip).
//   p_ij  = exp(z_ij - lse_i)            (recomputed from q, k and the saved log-sum)
//   ds_ij = p_ij * (dout_i.v_j - delta_i) * dz/ds,   delta_i = dout_i.o_i,   dz/ds = 1 - tanh^2 under a cap
//   dq_i  = scale * sum_j ds_ij k_j      dk_j = scale * sum_i ds_ij q_i      dv_j = sum_i p_ij dout_i
// Two passes over the score blocks, each writing every output row once from one workgroup: nothing is added atomically, so
// results do not depend on the order of workgroups (the price: 7 products where one pass with atomic adds takes 5).  Key heads
// that several query heads share sum over them inside the workgroup.
#include <algorithm>
#include <type_traits>

#include "kernels_seq.h"
#include "seq_attn.h"

namespace sttran {

// delta and the rows' key ranges: LPR lanes a (row, head), 16 bytes a lane, from (row, head) number `first` on.  The sums take out in
// full width: out + what its rounding took (out_lo), because delta's error is common to a whole row of ds
template <class T, int LPR>
__global__ void __launch_bounds__(256) seq_attn_delta_kernel(SeqAttnArgs A, int64_t first) {
  const int64_t item = first + ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
  const int c = threadIdx.x % LPR;
  if (item >= (int64_t)A.tq * A.hq) return;
  const int row = (int)(item / A.hq), head = (int)(item % A.hq), dbytes = A.d * (int)sizeof(T);
  const seq_u32x4 g = seq_row_chunk(A.raw[3].p + row * A.raw[3].t + head * A.raw[3].h, c, dbytes, A.aln);
  const seq_u32x4 o = seq_row_chunk(A.out + item * dbytes, c, dbytes, A.aln);
  seq_u32x4 r = {0, 0, 0, 0};
  if (A.out_lo) r = seq_row_chunk(A.out_lo + item * dbytes, c, dbytes, A.aln);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < SeqElt<T>::kPer16; ++i)
    s = fmaf(SeqElt<T>::get(g, i), SeqElt<T>::get(o, i) + (sizeof(T) == 2 ? SeqElt<T>::get(r, i) : 0.f), s);
  s = seq_group_sum<LPR>(s);
  if (c) return;
  A.delta[(int64_t)head * A.tq + row] = s;
  if (head == 0) {
    const SeqRow i = seq_row(A, row, seq_find(A.off_q, A.nseq, row));
    A.rows[row] = make_int4(i.lo, i.hi, i.base, 0);
  }
}

// p and ds of one pair from its products (s = q.k, dp = dout.v); hidden pairs become exact zeros in both
template <int CAP, bool SLOPE>
__device__ __forceinline__ void seq_pair(const SeqScore& sc, float& s, float& dp, bool seen, float lse, float delta, int away) {
  float z, bend = 1.f;
  if constexpr (CAP != kSeqCapNone) {
    const float t = seq_tanh<CAP == kSeqCapNear>(s * sc.mul);
    bend = 1.f - t * t;
    z = fmaf(sc.capl, t, -lse);
  } else {
    z = fmaf(s, sc.mul, -lse);
  }
  if constexpr (SLOPE) z = fmaf(-sc.slope, fabsf((float)away), z);
  const float p = __builtin_amdgcn_exp2f(z);
  dp = (dp - delta) * p;
  if constexpr (CAP != kSeqCapNone) dp *= bend;
  s = seen ? p : 0.f;
  dp = seen ? dp : 0.f;
}
__device__ __forceinline__ void seq_pair_any(const SeqAttnArgs& A, const SeqScore& sc, float& s, float& dp, bool seen, float lse, float delta,
                                             int away) {
  if (A.cap > 0.f) {
    if (A.slope) seq_pair<kSeqCap, true>(sc, s, dp, seen, lse, delta, away);
    else seq_pair<kSeqCap, false>(sc, s, dp, seen, lse, delta, away);
  } else {
    if (A.slope) seq_pair<kSeqCapNone, true>(sc, s, dp, seen, lse, delta, away);
    else seq_pair<kSeqCapNone, false>(sc, s, dp, seen, lse, delta, away);
  }
}
// ---- dq: own rows = queries, keys and values stream ---------------------------------------------------------------------
template <class C>
__device__ __forceinline__ void seq_attn_dq_again(const SeqAttnArgs& A, const SeqScore& sc, uint32_t rows, SeqRow me, int row0, int head, int dh) {
  using T = typename C::E;
  const int kvh = head / (A.hq / A.hk);
#pragma unroll 1
  for (int n = 0; n < 32; ++n) {
    const int row = row0 + n;
    if (!(rows >> n & 1) || row >= A.tq || n % C::DS != dh) continue;
    const int lo = __shfl(me.lo, n), hi = __shfl(me.hi, n), base = __shfl(me.base, n);
    const SeqSpread q = seq_spread<T>(A.raw[0].p + head * A.raw[0].h + (int64_t)row * A.raw[0].t, A.d);
    const SeqSpread g = seq_spread<T>(A.raw[3].p + head * A.raw[3].h + (int64_t)row * A.raw[3].t, A.d);
    const float lse = A.lse[(int64_t)head * A.tq + row], delta = A.delta[(int64_t)head * A.tq + row];
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int key = lo; key < hi; ++key) {
      const SeqSpread k = seq_spread<T>(A.raw[1].p + kvh * A.raw[1].h + (int64_t)key * A.raw[1].t, A.d);
      const SeqSpread v = seq_spread<T>(A.raw[2].p + kvh * A.raw[2].h + (int64_t)key * A.raw[2].t, A.d);
      float s = seq_spread_dot(q, k), dp = seq_spread_dot(g, v);
      seq_pair_any(A, sc, s, dp, true, lse, delta, base - key);
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = fmaf(dp, k.x[u], o[u]);
      if (!(dp == dp)) break;                        // all of the row is NaN, whatever follows
    }
    seq_spread_store<T>(A.dq + ((int64_t)row * A.hq + head) * A.d * C::OS, nullptr, o, A.scale, A.d);
  }
}

template <class C>
struct SeqDqLds {                                        // as SeqFwdLds, with two partial blocks a wave
  static constexpr int kBufs = C::DS == 1 ? 2 : 1;
  // the partial blocks go where the values' tile was (it is used up before them), where it is large enough
  static constexpr int kNeed = C::DS > 1 ? C::NW * SeqShare<C, 2>::kWave : 0;
  static constexpr bool kOver = C::DS > 1 && kNeed <= C::kTileBytes;
  static constexpr int kXch = kOver ? C::kTileBytes : 2 * kBufs * C::kTileBytes;
  static constexpr int kRed = 2 * kBufs * C::kTileBytes + (kOver ? 0 : kNeed), kBytes = kRed + C::NW * 8;
};
// Three products, bound as the forward pass.  Measured on the same sequences as there: 412 us, 960 TFLOP/s (bfloat16, 128 columns);
// 76 us (64 columns, short, ds with 16 bits: vector units busy 0.46, matrix pipe 0.18); 1520 us (fp32 on planes, 242 columns).
template <class C, int CAP, bool SLOPE, bool TWO>
__global__ void __launch_bounds__(C::NT) __attribute__((amdgpu_waves_per_eu(2, 2)))
seq_attn_dq_kernel(SeqAttnArgs A) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* xch = smem + SeqDqLds<C>::kXch;
  int* red = reinterpret_cast<int*>(smem + SeqDqLds<C>::kRed);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int tiles = (A.tq + C::RB - 1) / C::RB;
  const int id = seq_xcd_order(blockIdx.x, gridDim.x);
  const int head = id / tiles, tile = tiles - 1 - seq_spread_tile(A, id % tiles, tiles, A.hq);
  const int kvh = head / (A.hq / A.hk), dh = w % C::DS;
  const int row0 = tile * C::RB + 32 * (w / C::DS), row = row0 + (lane & 31);
  const int dbytes = C::row_bytes(A.d);

  SeqRow me{0, 0, 0};
  float lse = INFINITY, delta = 0.f;
  if (row < A.tq) {
    const int4 r = A.rows[row];
    me.lo = r.x; me.hi = r.y; me.base = r.z;
    lse = A.lse[(int64_t)head * A.tq + row];
    delta = A.delta[(int64_t)head * A.tq + row];
  }
  int lo = me.hi > me.lo ? me.lo : INT_MAX, hi = me.hi;
  seq_wave_range(lo, hi);
  const int wlo = lo, whi = hi;
  if (lane == 0) { red[2 * w] = lo; red[2 * w + 1] = hi; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < C::NW; ++i) { lo = min(lo, red[2 * i]); hi = max(hi, red[2 * i + 1]); }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  int beg = lo, end = max(hi, lo);
  if (hi <= 0) beg = end = 0;

  const char *kp = A.k + kvh * A.k_h, *vp = A.v + kvh * A.v_h;
  SeqMover mk, mv;
  mk.init<C>(A.k_t, dbytes);
  mv.init<C>(A.v_t, dbytes);
  char *kt_lds = smem, *vt_lds = smem + C::kTileBytes;
  if (beg < end) {
    seq_tile_move<C>(mk, kt_lds, kp, A.k_t, beg, end, dbytes);
    seq_tile_move<C>(mv, vt_lds, vp, A.v_t, beg, end, dbytes);
  }
  seq_u32x4 oq[C::PL * C::NF], og[C::PL * C::NF];
  seq_own_load<C>(oq, A.q + head * A.q_h, A.q_t, row0, A.tq, dh, dbytes);
  seq_own_load<C>(og, A.dout + head * A.do_h, A.do_t, row0, A.tq, dh, dbytes);
  const SeqScore sc(A, head);
  seq_f32x16 acc[C::NB];
#pragma unroll
  for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[nb][e] = 0.f;
  seq_tile_done<C>(mk, kt_lds, dbytes);
  seq_tile_done<C>(mv, vt_lds, dbytes);
  __syncthreads();

  for (int kt = beg, buf = 0; kt < end; kt += C::BR) {
    const bool more = kt + C::BR < end;
    char *kn = kt_lds, *vn = vt_lds;
    if constexpr (C::DS == 1) {
      kn = smem + (buf ^ 1) * 2 * C::kTileBytes;
      vn = kn + C::kTileBytes;
      if (more) {
        seq_tile_move<C>(mk, kn, kp, A.k_t, kt + C::BR, end, dbytes);
        seq_tile_move<C>(mv, vn, vp, A.v_t, kt + C::BR, end, dbytes);
      }
    }
#pragma unroll 1
    for (int u = 0; u < C::NSUB; ++u) {
      const int kb = kt + 32 * u;
      const bool active = wlo < min(kb + 32, end) && whi > kb;
      seq_f32x16 s, dp;
      if (active) {
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = 0.f;
        seq_scores<C>(dp, vt_lds, u, dh, og);
      }
      if constexpr (C::DS > 1) {                     // the keys' tile was still on its way while the values' was used
        if (kt > beg) seq_tile_done<C>(mk, kt_lds, dbytes);
        __syncthreads();
      }
      if (active) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
        seq_scores<C>(s, kt_lds, u, dh, oq);
      }
      if constexpr (C::DS > 1) {
        static_assert(C::NSUB == 1, "one pair of blocks is exchanged");
        if (active) {
          SeqShare<C, 2>::put(s, xch, w - dh, dh, 0);
          SeqShare<C, 2>::put(dp, xch, w - dh, dh, 1);
        }
        __syncthreads();                             // the values' tile is free
        if (!SeqDqLds<C>::kOver && more) seq_tile_move<C>(mv, vt_lds, vp, A.v_t, kt + C::BR, end, dbytes);
      }
      const bool full = __all(me.lo <= kb && me.hi >= kb + 32);
      if constexpr (C::DS == 1) {
        if (!active) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x = s[e], y = dp[e];
          seq_pair<CAP, SLOPE>(sc, x, y, true, lse, delta, me.base - kb - 4 * h - 8 * (e >> 2) - (e & 3));
          dp[e] = y;
        }
        if (!full) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = kb + 4 * h + 8 * (e >> 2) + (e & 3);
            dp[e] = key >= me.lo && key < me.hi ? dp[e] : 0.f;
          }
        }
      } else {
        // each wave of the team sums and finishes its share of the block's quads, then all take the whole
        using S = SeqShare<C, 2>;
        if (active) {
#pragma unroll
          for (int i = 0; i < S::GP; ++i) {
            const int g = dh * S::GP + i;
            const seq_f32x4 a = S::sum(s, xch, w - dh, dh, 0, i);
            seq_f32x4 b = S::sum(dp, xch, w - dh, dh, 1, i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = kb + 8 * g + 4 * h + e;
              float x = a[e], y = b[e];
              seq_pair<CAP, SLOPE>(sc, x, y, full || (key >= me.lo && key < me.hi), lse, delta, me.base - key);
              b[e] = y;
            }
            S::leave(b, xch, w - dh, dh, 1, i);
          }
        }
        __syncthreads();
        if (active) S::take(dp, xch, w - dh, 1);
        if constexpr (SeqDqLds<C>::kOver) {
          __syncthreads();                           // the blocks are read: the next values may come
          if (more) seq_tile_move<C>(mv, vt_lds, vp, A.v_t, kt + C::BR, end, dbytes);
        }
        if (!active) continue;
      }
      seq_reduce<C, TWO>(acc, kt_lds, u, dh, dp);
    }
    if (more) {
      if constexpr (C::DS == 1) seq_tile_done<C>(mk, kn, dbytes);
      seq_tile_done<C>(mv, vn, dbytes);
    }
    __syncthreads();
    if constexpr (C::DS == 1) {
      buf ^= 1;
      kt_lds = kn; vt_lds = vn;
    } else {
      if (more) seq_tile_move<C>(mk, kt_lds, kp, A.k_t, kt + C::BR, end, dbytes);
    }
  }
  const uint32_t bad = seq_bad_rows<C>(acc, 0, red);
  if (bad) seq_attn_dq_again<C>(A, sc, bad, me, row0, head, dh);
  if (row >= A.tq || (bad >> (lane & 31) & 1)) return;
  seq_store_own<C>(acc, A.scale, A.dq + ((int64_t)row * A.hq + head) * A.d * C::OS, nullptr, dh, A.d, A.aln);
}

// ---- dk, dv: own rows = keys, queries and dout stream ---------------------------------------------------------------------
// The work of a key tile -- (query head of the group, tile of query rows) in this order -- may be cut into A.splits shares of equal
// length, one workgroup each: i0 .. i1 here
template <class C>
__device__ __forceinline__ void seq_attn_dkv_again(const SeqAttnArgs& A, uint32_t rows, int row0, int kvh, int qbeg, int qend, int i0, int i1,
                                                   int dh, float* part) {
  using T = typename C::E;
  const int grp = A.hq / A.hk, nt = (qend - qbeg + C::BR - 1) / C::BR;
#pragma unroll 1
  for (int n = 0; n < 32; ++n) {
    const int key = row0 + n;
    if (!(rows >> n & 1) || key >= A.tk || n % C::DS != dh) continue;
    const SeqSpread k = seq_spread<T>(A.raw[1].p + kvh * A.raw[1].h + (int64_t)key * A.raw[1].t, A.d);
    const SeqSpread v = seq_spread<T>(A.raw[2].p + kvh * A.raw[2].h + (int64_t)key * A.raw[2].t, A.d);
    float dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
    bool rest = true;                                // false: all of dk's and dv's row is NaN, whatever follows
#pragma unroll 1
    for (int it = i0; it < i1 && rest; ++it) {
      const int head = kvh * grp + it / nt, q0 = qbeg + it % nt * C::BR, q1 = min(q0 + C::BR, qend);
      const SeqScore sc(A, head);
#pragma unroll 1
      for (int row = q0; row < q1 && rest; ++row) {
        const int4 r = A.rows[row];
        if (key < r.x || key >= r.y) continue;
        const SeqSpread q = seq_spread<T>(A.raw[0].p + head * A.raw[0].h + (int64_t)row * A.raw[0].t, A.d);
        const SeqSpread o = seq_spread<T>(A.raw[3].p + head * A.raw[3].h + (int64_t)row * A.raw[3].t, A.d);
        float s = seq_spread_dot(q, k), dp = seq_spread_dot(o, v);
        seq_pair_any(A, sc, s, dp, true, A.lse[(int64_t)head * A.tq + row], A.delta[(int64_t)head * A.tq + row], r.z - key);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          dk[u] = fmaf(dp, q.x[u], dk[u]);
          dv[u] = fmaf(s, o.x[u], dv[u]);
        }
        rest = s == s || dp == dp;
      }
    }
    const int64_t at = ((int64_t)key * A.hk + kvh) * A.d;
    if (part) {
      seq_spread_store<float>((char*)(part + at), nullptr, dk, A.scale, A.d);
      seq_spread_store<float>((char*)(part + (int64_t)A.tk * A.hk * A.d + at), nullptr, dv, 1.f, A.d);
    } else {
      seq_spread_store<T>(A.dk + at * C::OS, nullptr, dk, A.scale, A.d);
      seq_spread_store<T>(A.dv + at * C::OS, nullptr, dv, 1.f, A.d);
    }
  }
}

template <class C>
struct SeqDkvLds {                                       // tiles, statistics of the tile's rows, partial and whole score blocks
  // bfloat16 at 128 columns a wave: keys, values and both accumulators are 192 registers of the 256 that two waves a SIMD leave each,
  // too many next to a pair of blocks (spilled, the kernel took 2.4 ms on three sequences of 4000 .. 8000 rows, 8 heads, where it now
  // takes 0.7): the values' fragments are read from LDS instead
  static constexpr bool kPark = C::OS == 2 && C::DH == 128;
  static constexpr int kParked = kPark ? C::NF * 1024 : 0;          // bytes a wave
  static constexpr int kBufs = C::DS == 1 ? 2 : 1, kStat = 5 * C::BR * 4;
  static constexpr int kRows = 2 * kBufs * C::kTileBytes, kXch = kRows + kBufs * kStat;
  static constexpr int kRed = kXch + (C::DS > 1 ? C::NW * SeqShare<C, 2>::kWave : 0);
  static constexpr int kOwn = (kRed + C::NW * 8 + 15) / 16 * 16, kBytes = kOwn + C::NW * kParked;
};
// Four products.  Two accumulators and both stationary operands do not fit the registers, so LDS carries the values' fragments beside the
// streamed tiles: 40 KB a wave and 32 query rows, 2560 cycles of a CU's LDS for 2048 of its matrix pipes -- the bound.  Measured on the
// same sequences: 680 us, 780 TFLOP/s, and 40 us to join the shares; 138 us (64 columns, short, 16 bits: one wave a SIMD, which waits for
// 0.46 of its time); 2120 us (fp32 on planes, 242 columns).
template <class C, int CAP, bool SLOPE, bool TWO>
__global__ void __launch_bounds__(C::NT) __attribute__((amdgpu_waves_per_eu(2, 2)))
seq_attn_dkv_kernel(SeqAttnArgs A) {
  using L = SeqDkvLds<C>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* xch = smem + L::kXch;
  int* red = reinterpret_cast<int*>(smem + L::kRed);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int tiles = (A.tk + C::RB - 1) / C::RB, grp = A.hq / A.hk;
  const int id = seq_xcd_order(blockIdx.x, gridDim.x);
  const int kvh = id / tiles, tile = seq_spread_tile(A, id % tiles, tiles, A.hk), dh = w % C::DS;
  const int first = tile * C::RB, row0 = first + 32 * (w / C::DS), key = row0 + (lane & 31);
  const int dbytes = C::row_bytes(A.d);

  // query rows that may see a key of this tile: those of the sequences that the tile touches
  int qbeg = 0, qend = 0;
  {
    const int s0 = seq_find_wave(A.off_k, A.nseq, first), s1 = min(seq_find_wave(A.off_k, A.nseq, min(first + C::RB, A.tk) - 1), A.nseq - 1);
    if (s0 < A.nseq) {
      qbeg = A.off_q[s0];
      qend = min(max(A.off_q[s1 + 1], 0), A.tq);
      const int at = max(first - A.off_k[s0], 0);
      if (A.causal && !(A.prefix && A.prefix[s0] > at)) {
        const int lq = A.off_q[s0 + 1] - qbeg, lk = A.off_k[s0 + 1] - A.off_k[s0];
        qbeg += min(max(at - (lk - lq), 0), max(lq, 0));
      }
      qbeg = min(max(qbeg, 0), A.tq);
    }
    qbeg = __builtin_amdgcn_readfirstlane(qbeg);
    qend = __builtin_amdgcn_readfirstlane(qend);
  }
  const int nt = (qend - qbeg + C::BR - 1) / C::BR;
  int i0 = 0, i1 = qbeg < qend ? grp * nt : 0;
  if (A.splits > 1) {
    const int64_t all = i1;
    i0 = (int)(all * blockIdx.y / A.splits);
    i1 = (int)(all * (blockIdx.y + 1) / A.splits);
  }

  SeqMover mq, mg;
  mq.init<C>(A.q_t, dbytes);
  mg.init<C>(A.do_t, dbytes);
  // backwards, so that the workgroups of a head's key tiles, which see different first rows where the order masks but the same last
  // ones, read the same tiles at the same time (a training step of three sequences of 4000 .. 8000 rows, 8 heads over 2, 128 columns,
  // 1740 -> 1619 us)
  int head = kvh * grp, row = qbeg;
  if (i0 < i1) {
    head += (i1 - 1) / nt;
    row += (i1 - 1) % nt * C::BR;
  }
  float sf[2];
  int4 si;
  const auto load_stat = [&](int head, int row) {         // threads tid < BR: their row's statistics
    const int r = row + tid;
    sf[0] = INFINITY; sf[1] = 0.f; si = make_int4(0, 0, 0, 0);
    if (tid < C::BR && r < qend) {
      const int64_t at = (int64_t)head * A.tq + r;
      sf[0] = A.lse[at]; sf[1] = A.delta[at]; si = A.rows[r];
    }
  };
  const auto store_stat = [&](char* to) {                 // [lse | delta | lo | hi | base][BR]
    if (tid < C::BR) {
      float* f = reinterpret_cast<float*>(to);
      int* n = reinterpret_cast<int*>(to);
      f[tid] = sf[0]; f[C::BR + tid] = sf[1];
      n[2 * C::BR + tid] = si.x; n[3 * C::BR + tid] = si.y; n[4 * C::BR + tid] = si.z;
    }
  };

  char *qt_lds = smem, *gt_lds = smem + C::kTileBytes, *st = smem + L::kRows;
  if (i0 < i1) {
    seq_tile_move<C>(mq, qt_lds, A.q + head * A.q_h, A.q_t, row, qend, dbytes);
    seq_tile_move<C>(mg, gt_lds, A.dout + head * A.do_h, A.do_t, row, qend, dbytes);
    load_stat(head, row);
    store_stat(st);
  }
  seq_u32x4 ok[C::PL * C::NF], ov[C::PL * C::NF];
  seq_own_load<C>(ok, A.k + kvh * A.k_h, A.k_t, row0, A.tk, dh, dbytes);
  seq_own_load<C>(ov, A.v + kvh * A.v_h, A.v_t, row0, A.tk, dh, dbytes);
  char* parked = smem + L::kOwn + w * L::kParked;       // read by this wave alone
  if constexpr (L::kPark) {
#pragma unroll
    for (int f = 0; f < C::NF; ++f) *reinterpret_cast<seq_u32x4*>(parked + f * 1024 + lane * 16) = ov[f];
  }
  seq_f32x16 dk[C::NB], dv[C::NB];
#pragma unroll
  for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
    for (int e = 0; e < 16; ++e) { dk[nb][e] = 0.f; dv[nb][e] = 0.f; }
  seq_tile_done<C>(mq, qt_lds, dbytes);
  seq_tile_done<C>(mg, gt_lds, dbytes);
  __syncthreads();

  for (int left = i1 - i0, buf = 0; left > 0; --left) {
    const bool more = left > 1;
    const SeqScore sc(A, head);
    row -= C::BR;                                    // the next tile's from here on
    if (row < qbeg) {
      --head;
      row = qbeg + (nt - 1) * C::BR;
    }
    char *qn = qt_lds, *gn = gt_lds, *sn = st;
    if constexpr (C::DS == 1) {
      qn = smem + (buf ^ 1) * 2 * C::kTileBytes;
      gn = qn + C::kTileBytes;
      sn = smem + L::kRows + (buf ^ 1) * L::kStat;
    }
    if (more) {
      load_stat(head, row);
      if constexpr (C::DS == 1) {
        seq_tile_move<C>(mq, qn, A.q + head * A.q_h, A.q_t, row, qend, dbytes);
        seq_tile_move<C>(mg, gn, A.dout + head * A.do_h, A.do_t, row, qend, dbytes);
      }
    }
    const float* rowf = reinterpret_cast<const float*>(st);
    const int* rowi = reinterpret_cast<const int*>(st) + 2 * C::BR;
    // p and ds of quad g of block u in place of its products
    const auto quad = [&](int u, int g, seq_f32x4& s4, seq_f32x4& p4) __attribute__((always_inline)) {
      const int at = 32 * u + 8 * g + 4 * h;
      const seq_f32x4 l4 = *reinterpret_cast<const seq_f32x4*>(rowf + at), d4 = *reinterpret_cast<const seq_f32x4*>(rowf + C::BR + at);
      int ba[4] = {0, 0, 0, 0};
      if constexpr (SLOPE) {
        const int4 b4 = *reinterpret_cast<const int4*>(rowi + 2 * C::BR + at);
        ba[0] = b4.x; ba[1] = b4.y; ba[2] = b4.z; ba[3] = b4.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = s4[i], y = p4[i];
        seq_pair<CAP, SLOPE>(sc, x, y, true, l4[i], d4[i], ba[i] - key);
        s4[i] = x; p4[i] = y;
      }
    };
    const auto hide = [&](int u, int g, seq_f32x4& s4, seq_f32x4& p4) __attribute__((always_inline)) {
      const int at = 32 * u + 8 * g + 4 * h;
      const int4 lo4 = *reinterpret_cast<const int4*>(rowi + at), hi4 = *reinterpret_cast<const int4*>(rowi + C::BR + at);
      const int lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool seen = key >= lo[i] && key < hi[i];
        s4[i] = seen ? s4[i] : 0.f;
        p4[i] = seen ? p4[i] : 0.f;
      }
    };
#pragma unroll 1
    for (int u = 0; u < C::NSUB; ++u) {
      const int rl = rowi[32 * u + (lane & 31)], rh = rowi[C::BR + 32 * u + (lane & 31)];
      const bool active = __any(rl < row0 + 32 && rh > row0), full = __all(rl <= row0 && rh >= row0 + 32);
      seq_f32x16 s, dp;
      if (active) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
        seq_scores<C>(s, qt_lds, u, dh, ok);
      }
      if constexpr (C::DS > 1) {                     // dout's tile was still on its way while q's was used
        if (left < i1 - i0) {
          seq_tile_done<C>(mg, gt_lds, dbytes);
          __syncthreads();
        }
      }
      if (active) {
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = 0.f;
        if constexpr (L::kPark) seq_scores_parked<C>(dp, gt_lds, u, dh, parked);
        else seq_scores<C>(dp, gt_lds, u, dh, ov);
      }
      if constexpr (C::DS == 1) {
        if (!active) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          seq_f32x4 a = seq_quad(s, g), b = seq_quad(dp, g);
          quad(u, g, a, b);
          seq_set_quad(s, g, a);
          seq_set_quad(dp, g, b);
          __builtin_amdgcn_sched_barrier(0);         // or all the quads' statistics are fetched at once
        }
        if (!full) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            seq_f32x4 a = seq_quad(s, g), b = seq_quad(dp, g);
            hide(u, g, a, b);
            seq_set_quad(s, g, a);
            seq_set_quad(dp, g, b);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        seq_reduce<C, TWO>(dv, gt_lds, u, dh, s);
        seq_reduce<C, TWO>(dk, qt_lds, u, dh, dp);
      } else {
        // each wave of the team sums and finishes its share of the block's quads, then all take the whole
        static_assert(C::NSUB == 1, "one pair of blocks is exchanged");
        using S = SeqShare<C, 2>;
        if (active) {
          S::put(s, xch, w - dh, dh, 0);
          S::put(dp, xch, w - dh, dh, 1);
        }
        __syncthreads();
        if (active) {
#pragma unroll
          for (int i = 0; i < S::GP; ++i) {
            const int g = dh * S::GP + i;
            seq_f32x4 a = S::sum(s, xch, w - dh, dh, 0, i), b = S::sum(dp, xch, w - dh, dh, 1, i);
            quad(u, g, a, b);
            if (!full) hide(u, g, a, b);
            S::leave(a, xch, w - dh, dh, 0, i);
            S::leave(b, xch, w - dh, dh, 1, i);
          }
        }
        __syncthreads();                             // also: the statistics' last reader has passed
        if (more) store_stat(st);
        if (active) {
          S::take(dp, xch, w - dh, 1);
          seq_reduce<C, TWO>(dk, qt_lds, u, dh, dp);
        }
        __syncthreads();                             // q's tile is free
        if (more) seq_tile_move<C>(mq, qt_lds, A.q + head * A.q_h, A.q_t, row, qend, dbytes);
        if (active) {
          S::take(s, xch, w - dh, 0);
          seq_reduce<C, TWO>(dv, gt_lds, u, dh, s);
        }
      }
    }
    if (more) {
      seq_tile_done<C>(mq, qn, dbytes);
      if constexpr (C::DS == 1) {
        seq_tile_done<C>(mg, gn, dbytes);
        store_stat(sn);
      }
    }
    __syncthreads();
    if constexpr (C::DS == 1) {
      buf ^= 1;
      qt_lds = qn; gt_lds = gn; st = sn;
    } else {
      if (more) seq_tile_move<C>(mg, gt_lds, A.dout + head * A.do_h, A.do_t, row, qend, dbytes);
    }
  }
  uint32_t bad = seq_bad_rows<C>(dk, 0, red);
  bad = seq_bad_rows<C>(dv, bad, red);
  float* part = A.splits > 1 ? A.part + 2 * blockIdx.y * ((int64_t)A.tk * A.hk * A.d) : nullptr;
  if (bad) seq_attn_dkv_again<C>(A, bad, row0, kvh, qbeg, qend, i0, i1, dh, part);
  if (key >= A.tk || (bad >> (lane & 31) & 1)) return;
  if (part) {
    const int64_t to = ((int64_t)key * A.hk + kvh) * A.d;
    seq_store_part<C>(dk, A.scale, part + to, dh, A.d, 4);
    seq_store_part<C>(dv, 1.f, part + (int64_t)A.tk * A.hk * A.d + to, dh, A.d, 4);
    return;
  }
  const int64_t at = ((int64_t)key * A.hk + kvh) * A.d * C::OS;
  seq_store_own<C>(dk, A.scale, A.dk + at, nullptr, dh, A.d, A.aln);
  seq_store_own<C>(dv, 1.f, A.dv + at, nullptr, dh, A.d, A.aln);
}

// dk, dv from the shares' partial sums, in the order of the shares: four elements a thread (n: elements of one of them)
template <class T>
__global__ void __launch_bounds__(256) seq_attn_dkv_join_kernel(SeqAttnArgs A, int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int left = (int)min((int64_t)4, n - i);
  const float* p = A.part + blockIdx.y * n + i;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < A.splits; ++s, p += 2 * n) {
    const seq_u32x4 r = seq_load16((const char*)p, 4 * left, 4);
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] += __uint_as_float(r[u]);
  }
  T* out = reinterpret_cast<T*>(blockIdx.y ? A.dv : A.dk) + i;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (u < left) out[u] = (T)x[u];
}

template <class C, int CAP, bool SLOPE, bool TWO>
static hipError_t dq_as(hipStream_t s, const SeqAttnArgs& A) {
  constexpr int lds = SeqDqLds<C>::kBytes;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  static DeviceMarks marks;
  auto fn = seq_attn_dq_kernel<C, CAP, SLOPE, TWO>;
  hipError_t e = marks.raise_lds(reinterpret_cast<const void*>(fn), lds);
  if (e != hipSuccess) return e;
  fn<<<(unsigned)((A.tq + C::RB - 1) / C::RB * A.hq), C::NT, lds, s>>>(A);
  return hipGetLastError();
}
template <class C, int CAP, bool SLOPE, bool TWO>
static hipError_t dkv_as(hipStream_t s, const SeqAttnArgs& A) {
  constexpr int lds = SeqDkvLds<C>::kBytes;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  static DeviceMarks marks;
  auto fn = seq_attn_dkv_kernel<C, CAP, SLOPE, TWO>;
  hipError_t e = marks.raise_lds(reinterpret_cast<const void*>(fn), lds);
  if (e != hipSuccess) return e;
  fn<<<dim3((unsigned)((A.tk + C::RB - 1) / C::RB * A.hk), (unsigned)A.splits), C::NT, lds, s>>>(A);
  e = hipGetLastError();
  if (e != hipSuccess || A.splits == 1) return e;
  const int64_t n = (int64_t)A.tk * A.hk * A.d;
  seq_attn_dkv_join_kernel<typename C::E><<<dim3((unsigned)((n + 1023) / 1024), 2), 256, 0, s>>>(A, n);
  return hipGetLastError();
}
// kernels by cap and distances as in the forward pass (same sequences: dq 440 -> 413 us, dk and dv 1180 -> 850 us)
template <class C, bool TWO = false>
static hipError_t dq(hipStream_t s, const SeqAttnArgs& A) {
  if constexpr (C::OS == 2) {
    if (A.cap > kSeqNearCap) return dq_as<C, kSeqCap, true, true>(s, A);
  }
  constexpr int cap = C::OS == 2 ? kSeqCapNear : kSeqCap;
  if (A.cap > 0.f) return A.slope ? dq_as<C, cap, true, TWO>(s, A) : dq_as<C, cap, false, TWO>(s, A);
  return A.slope ? dq_as<C, kSeqCapNone, true, TWO>(s, A) : dq_as<C, kSeqCapNone, false, TWO>(s, A);
}
template <class C, bool TWO = false>
static hipError_t dkv(hipStream_t s, const SeqAttnArgs& A) {
  if constexpr (C::OS == 2) {
    if (A.cap > kSeqNearCap) return dkv_as<C, kSeqCap, true, true>(s, A);
  }
  constexpr int cap = C::OS == 2 ? kSeqCapNear : kSeqCap;
  if (A.cap > 0.f) return A.slope ? dkv_as<C, cap, true, TWO>(s, A) : dkv_as<C, cap, false, TWO>(s, A);
  return A.slope ? dkv_as<C, kSeqCapNone, true, TWO>(s, A) : dkv_as<C, kSeqCapNone, false, TWO>(s, A);
}
// 64 lanes for each of 2^26 wide rows are more threads than a launch may have: 2^31 a launch.  (Threads that walk on by the grid instead
// cost a training step more: 96 sequences of 37 .. 500 rows 309.5 -> 311.3 us, three of 3000 .. 8192 rows 1456 -> 1463.)
template <class T, int LPR>
static hipError_t delta_as(hipStream_t s, const SeqAttnArgs& A) {
  constexpr int64_t most = (int64_t(1) << 31) / LPR;
  const int64_t items = (int64_t)A.tq * A.hq;
  for (int64_t first = 0; first < items; first += most) {
    seq_attn_delta_kernel<T, LPR><<<(unsigned)((std::min(items - first, most) * LPR + 255) / 256), 256, 0, s>>>(A, first);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
template <class T>
static hipError_t delta(hipStream_t s, const SeqAttnArgs& A) {
  const int chunks = (A.d * (int)sizeof(T) + 15) / 16;
  if (chunks <= 8) return delta_as<T, 8>(s, A);
  if (chunks <= 16) return delta_as<T, 16>(s, A);
  if (chunks <= 32) return delta_as<T, 32>(s, A);
  return delta_as<T, 64>(s, A);
}

template <class T, bool VEC, bool TWO>
static hipError_t pick_dq(hipStream_t s, const SeqAttnArgs& A) {
  if (A.d <= 64) return dq<SeqTile<T, 64, 1, 2, 64, VEC>, TWO>(s, A);
  if (A.d <= 128) return dq<SeqTile<T, 128, sizeof(T) == 2 ? 1 : 2, 4, sizeof(T) == 2 ? 64 : 32, VEC>, TWO>(s, A);
  return dq<SeqTile<T, 256, sizeof(T) == 2 ? 2 : 4, 4, 32, VEC>, sizeof(T) == 2>(s, A);
}
// Waves a workgroup with 64 columns: two in bfloat16 (a training step of 96 sequences of 37 .. 500 rows 313 -> 301 us; 64 x 256 rows,
// 8 heads over 2, 174 -> 164; 1 x 16384 1942 -> 1967), four in fp32 (128 x 128 rows 311 us, with two 372)
template <class T, bool VEC, bool TWO>
static hipError_t pick_dkv(hipStream_t s, const SeqAttnArgs& A) {
  if (A.d <= 64) return dkv<SeqTile<T, 64, 1, sizeof(T) == 2 ? 2 : 4, 64, VEC>, TWO>(s, A);
  if (A.d <= 128) return dkv<SeqTile<T, 128, sizeof(T) == 2 ? 1 : 2, 4, 32, VEC>, TWO>(s, A);
  return dkv<SeqTile<T, 256, 4, sizeof(T) == 2 ? 4 : 8, 32, VEC>, sizeof(T) == 2>(s, A);
}
static hipError_t pick_dq_planes(hipStream_t s, const SeqAttnArgs& A) {
  if (A.d <= 64) return dq<SeqTile<float, 64, 1, 4, 32, true, 3>>(s, A);
  if (A.d <= 128) return dq<SeqTile<float, 128, 2, 4, 32, true, 3>>(s, A);
  return dq<SeqTile<float, 256, 4, 8, 32, true, 3>>(s, A);
}
static hipError_t pick_dkv_planes(hipStream_t s, const SeqAttnArgs& A) {
  if (A.d <= 64) return dkv<SeqTile<float, 64, 1, 4, 32, true, 3>>(s, A);
  if (A.d <= 128) return dkv<SeqTile<float, 128, 2, 4, 32, true, 3>>(s, A);
  return dkv<SeqTile<float, 256, 4, 8, 32, true, 3>>(s, A);
}
int seq_attn_dkv_tile(int bf16, bool planes, int d) {
  if (planes) return d <= 64 ? 128 : 64;
  if (d <= 64) return bf16 ? 64 : 128;
  return d > 128 ? (bf16 ? 32 : 64) : bf16 ? 128 : 64;
}

// bfloat16 in sequences of fewer than 512 rows on average, or of more than 128 columns: p and ds enter the products with 16 bits (TWO).
// With 8, dq and dk carry that rounding, the forward pass's (in delta) and the result's own: 1.44 .. 1.49 times the error of the last
// alone, but up to 1.97 where few terms sum (1 .. 60 rows) and 1.54 with 242 columns; with 16 bits 1.02 .. 1.13.  The price, a training
// step: 96 sequences of 37 .. 500 rows 285 -> 312 us; 8 x 2048 rows of 242 columns 1972 -> 2048; three of 4000 .. 8000 rows of 128 columns,
// 1663 -> 1855, keep 8.  Rows at odd 2 bytes take 16 bits always.
hipError_t launch_seq_attn_bwd(hipStream_t s, int bf16, bool planes, const SeqAttnArgs& A) {
  const bool vec = A.aln >= 4, two = A.d > 128 || seq_fewer_rows(A, 512);
  if (A.tq > 0) {
    hipError_t e = bf16 ? delta<__bf16>(s, A) : delta<float>(s, A);
    if (e != hipSuccess) return e;
    if (planes) e = pick_dq_planes(s, A);
    else if (bf16) e = !vec ? pick_dq<__bf16, false, true>(s, A) : two ? pick_dq<__bf16, true, true>(s, A) : pick_dq<__bf16, true, false>(s, A);
    else e = pick_dq<float, true, false>(s, A);                // 4-byte elements are 4-byte aligned
    if (e != hipSuccess) return e;
  }
  if (A.tk == 0) return hipSuccess;
  if (planes) return pick_dkv_planes(s, A);
  if (bf16) return !vec ? pick_dkv<__bf16, false, true>(s, A) : two ? pick_dkv<__bf16, true, true>(s, A) : pick_dkv<__bf16, true, false>(s, A);
  return pick_dkv<float, true, false>(s, A);
}

}  // namespace sttran
