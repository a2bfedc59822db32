// seq_attn.h -- what the forward and backward kernels of attention over packed sequences share (kernels_seq_attn.hip,
// kernels_seq_attn_bwd.hip).
//
// One scheme for every product.  A wave owns 32 STATIONARY rows (queries; keys in the dk/dv kernel), one per lane column of a
// 32x32 matrix-instruction block, held in registers as the B operand.  The other side STREAMS through LDS in tiles of BR rows.
//   scores      S[stream row][own row] = sum_d X[stream row][d] Y[own row][d]      A = tile rows as they lie (16-byte reads)
//   reductions  Z[d][own row] += sum_r W[r][d] P[r][own row]                       A = tile columns (transposed reads), B = P
// The accumulator layout of the score block (lane = own row, 16 registers = stream rows) IS the B layout of the second product
// once the contraction index is permuted, so probabilities go from the exponential into the next matrix instruction without
// leaving their lane; row statistics of an own row live in one lane (plus its partner 32 lanes further).
// bfloat16: v_mfma_f32_32x32x16_bf16, transposed reads by ds_read_b64_tr_b16; fp32: v_mfma_f32_32x32x2_f32 (exact products), or
// (PL = 3, sequences of some hundred keys) three bfloat16 planes: x = hi + mid + lo, 8 bits of mantissa each, so the sum is x exactly,
// and of the nine products of two such numbers the six that are not below 2^-24 of the largest, each exact in the fp32 accumulator.
// That is 6 / 16 of the exact instruction's time, and leaves the vector units free meanwhile, which fp32 matrix instructions do not.
// Head dims are padded to DP = 64 / 128 / 256 with zeros.  Where 32 own rows and their accumulators would not fit half of a SIMD's
// registers (so that two waves share it), a team of DS = 2 or 4 waves shares 32 own rows, each contracting (scores) and accumulating
// (reductions) its part of d; the partial scores meet in LDS.
#pragma once
#include <type_traits>

#include "seq_common.h"

namespace sttran {

template <class T, int DP_, int DS_, int NW_, int BR_, bool VEC_, int PL_ = 1>
struct SeqTile {
  using E = T;                                       // what the caller's tensors hold
  static constexpr bool VEC = VEC_;
  static constexpr int DP = DP_, DS = DS_, NW = NW_, BR = BR_;
  static constexpr int PL = PL_;                     // 3: fp32 as three bfloat16 planes
  static constexpr int OS = sizeof(T), ES = PL == 3 ? 2 : OS;      // bytes of an element of the tensors / of a tile
  static constexpr int NT = NW * 64;                 // threads
  static constexpr int DH = DP / DS;                 // columns of one wave
  static constexpr int RS = DP * ES;                 // bytes of a tile row
  static constexpr int NC = RS / 16;                 // 16-byte chunks of a tile row
  static constexpr int NF = DH * ES / 32;            // fragments (16 bytes a lane) of one own row's part, a plane
  static constexpr int NB = DH / 32;                 // 32-column blocks of one wave's accumulator
  static constexpr int NSUB = BR / 32;
  static constexpr int RB = 32 * NW / DS;            // own rows of a workgroup
  static constexpr int NL = BR * NC / NT;            // chunks a thread moves per tile and plane
  static constexpr int kPlaneBytes = BR * RS, kTileBytes = PL * kPlaneBytes;
  static __host__ __device__ int row_bytes(int d) { return PL == 3 ? (d + 7) / 8 * 16 : d * OS; }      // of a plane's row in memory
  static constexpr int kStep = NT / NC;              // tile rows between a thread's chunks
  static_assert(BR * NC % NT == 0 && NT % NC == 0, "whole chunks");
  static_assert(2 * kStep % (ES == 4 ? 8 : 16) == 0, "two source offsets: the layout's XOR repeats every 8 (fp32) or 16 rows");
};

// chunk position of (row, chunk): an XOR that spreads both access patterns over the banks -- eight consecutive rows at one
// chunk (16-byte reads of the scores) and four consecutive rows at one or two neighbouring chunks (transposed reads)
template <class C>
__device__ __forceinline__ int seq_swz(int row) {
  if constexpr (C::NC == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else if constexpr (C::ES == 2) return ((row & 3) << 2) | ((row >> 2) & 3);
  else return (row & 7) | (((row >> 2) & 1) << 3);
}

// ---- loads.  VEC (addresses and row lengths divisible by 4): buffer loads, whose bounds check -- dword by dword -- turns rows from
// `hi` on into zeros (nothing there is read, so what lies behind the last sequence cannot reach a sum); what a row's last chunk
// reads behind the row's end is masked off.  Otherwise (odd head dims of 2-byte elements): element by element.
constexpr uint32_t kSeqOob = 0x80000000u;
__device__ __forceinline__ auto seq_rsrc(const char* base, int64_t stride, int rows, int dbytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, rows > 0 ? (int)((rows - 1) * stride + dbytes) : 0, 0x00027000);
}
// masks of the four dwords of chunk c: all ones within the row
__device__ __forceinline__ seq_u32x4 seq_chunk_mask(int c, int dbytes) {
  seq_u32x4 m;
#pragma unroll
  for (int u = 0; u < 4; ++u) m[u] = 16 * c + 4 * u < dbytes ? 0xffffffffu : 0u;
  return m;
}

// Moving tiles.  VEC: straight from memory into LDS (16 bytes a lane, no registers), lane i of a wave to 16 i behind the wave's
// base; the XOR of the layout is applied to the SOURCE chunk.  A tile's mover is done with seq_tile_done: its own loads have
// landed and the tail of a row that is no multiple of 16 bytes is cleared (a load reads on behind the row there); a barrier then
// shows the tile to the others.  The copy into a tile may only start behind a barrier that every reader of its old content passed.
struct SeqMover {
  uint32_t off[2];                                  // source offset of an even / odd chunk's row and chunk, or kSeqOob
  uint32_t tail;                                    // bit i: this thread moves the last, partial chunk in its i-th row
  int wave;
  template <class C>
  __device__ __forceinline__ void init(int64_t stride, int dbytes) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    tail = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = threadIdx.x / C::NC + i * C::kStep, c = (threadIdx.x % C::NC) ^ seq_swz<C>(row);
      off[i] = 16 * c < dbytes ? (threadIdx.x / C::NC) * (uint32_t)stride + 16 * c : kSeqOob;
      if ((dbytes & 15) && c == dbytes >> 4) tail |= 1u << i;
    }
  }
};
template <class C>
__device__ __forceinline__ void seq_tile_move(const SeqMover& mv, char* tile, const char* base, int64_t stride, int row0, int hi, int dbytes) {
#ifdef __HIP_DEVICE_COMPILE__                              // the host pass refuses 16-byte copies into LDS
  const int rows = min(hi - row0, C::BR);
  if constexpr (C::VEC) {
#pragma unroll
    for (int pl = 0; pl < C::PL; ++pl) {                 // a row of planes is [plane][d, padded to 8] in memory
      const auto rs = seq_rsrc(base + (int64_t)row0 * stride + pl * dbytes, stride, rows, dbytes);
#pragma unroll
      for (int i = 0; i < C::NL; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(tile + pl * C::kPlaneBytes + (i * C::NT + mv.wave * 64) * 16),
                                                 16, mv.off[i & 1], i * C::kStep * (uint32_t)stride, 0, 0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < C::NL; ++i) {
      const int row = threadIdx.x / C::NC + i * C::kStep, c = threadIdx.x % C::NC;
      const seq_u32x4 r = seq_load16(base + (int64_t)(row0 + row) * stride + 16 * c, row < rows ? dbytes - 16 * c : 0, 2);
      *reinterpret_cast<seq_u32x4*>(tile + row * C::RS + ((c ^ seq_swz<C>(row)) << 4)) = r;
    }
  }
#endif
}
template <class C>
__device__ __forceinline__ void seq_tile_done(const SeqMover& mv, char* tile, int dbytes) {
  if constexpr (C::VEC) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (dbytes & 15) {
#pragma unroll
      for (int i = 0; i < C::NL; ++i)
        if (mv.tail >> (i & 1) & 1) {
          uint32_t* p = reinterpret_cast<uint32_t*>(tile + (i * C::NT + threadIdx.x) * 16);
          if ((dbytes & 15) <= 4) p[1] = 0;
          if ((dbytes & 15) <= 8) p[2] = 0;
          p[3] = 0;
        }
    }
  }
}

// own rows row0 .. row0 + 31 of this wave as B fragments, plane behind plane
template <class C>
__device__ __forceinline__ void seq_own_load(seq_u32x4 (&f)[C::PL * C::NF], const char* base, int64_t stride, int row0, int rows, int dh, int dbytes) {
  const int h = (threadIdx.x >> 5) & 1, n = threadIdx.x & 31, c0 = dh * (C::DH * C::ES / 16) + h;
  const int left = min(rows - row0, 32);
  const char* p = base + (int64_t)row0 * stride;
  if constexpr (C::VEC) {
#pragma unroll
    for (int pl = 0; pl < C::PL; ++pl) {
      const auto rs = seq_rsrc(p + pl * dbytes, stride, left, dbytes);
#pragma unroll
      for (int i = 0; i < C::NF; ++i) {
        const int at = 16 * (c0 + 2 * i);
        f[pl * C::NF + i] =
            __builtin_bit_cast(seq_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at < dbytes ? n * (uint32_t)stride + at : kSeqOob, 0, 0));
      }
    }
#pragma unroll
    for (int i = 0; i < C::PL * C::NF; ++i) f[i] &= seq_chunk_mask(c0 + 2 * (i % C::NF), dbytes);
  } else {
#pragma unroll
    for (int i = 0; i < C::NF; ++i) {
      const int c = c0 + 2 * i;
      f[i] = seq_load16(p + (int64_t)n * stride + 16 * c, n < left ? dbytes - 16 * c : 0, 2);
    }
  }
}

// smallest lo and largest hi over the lanes of a wave
__device__ __forceinline__ void seq_wave_range(int& lo, int& hi) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    lo = min(lo, __shfl_xor(lo, o));
    hi = max(hi, __shfl_xor(hi, o));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
}

__device__ __forceinline__ seq_f32x16 seq_mma(seq_f32x16 acc, seq_u32x4 a, seq_u32x4 b) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(seq_bf16x8, a), __builtin_bit_cast(seq_bf16x8, b), acc, 0, 0, 0);
}
// (a0 + a1 + a2)(b0 + b1 + b2) without the three smallest terms, small ones first
__device__ __forceinline__ seq_f32x16 seq_six(seq_f32x16 acc, seq_u32x4 a0, seq_u32x4 a1, seq_u32x4 a2, seq_u32x4 b0, seq_u32x4 b1, seq_u32x4 b2) {
  acc = seq_mma(acc, a2, b0);
  acc = seq_mma(acc, a0, b2);
  acc = seq_mma(acc, a1, b1);
  acc = seq_mma(acc, a1, b0);
  acc = seq_mma(acc, a0, b1);
  return seq_mma(acc, a0, b0);
}
// x = hi + mid + lo, each a bfloat16 (what the rounding of one leaves is the next one's number)
__device__ __forceinline__ void seq_split3(float x, __bf16& hi, __bf16& mid, __bf16& lo) {
  hi = (__bf16)x;
  const float r = x - (float)hi;
  mid = (__bf16)r;
  lo = (__bf16)(r - (float)mid);
}

// acc[stream row][own row] += tile . own
template <class C>
__device__ __forceinline__ void seq_scores(seq_f32x16& acc, const char* tile, int sub, int dh, const seq_u32x4 (&own)[C::PL * C::NF]) {
  const int lane = threadIdx.x & 63, row = 32 * sub + (lane & 31), h = lane >> 5;
  const char* p = tile + row * C::RS;
  const int x = (h ^ seq_swz<C>(row)) << 4;
#pragma unroll
  for (int f = 0; f < C::NF; ++f) {
    const seq_u32x4 a = *reinterpret_cast<const seq_u32x4*>(p + ((dh * C::DH * C::ES + 32 * f) ^ x));
    if constexpr (C::PL == 3) {
      const seq_u32x4 a1 = *reinterpret_cast<const seq_u32x4*>(p + C::kPlaneBytes + ((dh * C::DH * C::ES + 32 * f) ^ x));
      const seq_u32x4 a2 = *reinterpret_cast<const seq_u32x4*>(p + 2 * C::kPlaneBytes + ((dh * C::DH * C::ES + 32 * f) ^ x));
      acc = seq_six(acc, a, a1, a2, own[f], own[C::NF + f], own[2 * C::NF + f]);
    } else if constexpr (C::ES == 2) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(seq_bf16x8, a), __builtin_bit_cast(seq_bf16x8, own[f]), acc, 0, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[u]), __uint_as_float(own[f][u]), acc, 0, 0, 0);
    }
  }
}

// the same with the own rows' fragments parked in LDS (`parked`: this wave's, fragment by fragment, 16 bytes a lane)
template <class C>
__device__ __forceinline__ void seq_scores_parked(seq_f32x16& acc, const char* tile, int sub, int dh, const char* parked) {
  const int lane = threadIdx.x & 63, row = 32 * sub + (lane & 31), h = lane >> 5;
  const char* p = tile + row * C::RS;
  const int x = (h ^ seq_swz<C>(row)) << 4;
#pragma unroll
  for (int f = 0; f < C::NF; ++f) {
    const seq_u32x4 a = *reinterpret_cast<const seq_u32x4*>(p + ((dh * C::DH * C::ES + 32 * f) ^ x));
    const seq_u32x4 b = *reinterpret_cast<const seq_u32x4*>(parked + f * 1024 + lane * 16);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(seq_bf16x8, a), __builtin_bit_cast(seq_bf16x8, b), acc, 0, 0, 0);
  }
}

// acc[d][own row] += tile^T . w, w = a score block's registers.  bfloat16: w is rounded to 8 bits of mantissa here, the one
// rounding of probabilities (or of their derivatives) on the way into the matrix instruction -- TWO: what that takes away follows in
// an instruction of its own, 16 bits in all; sums stay in fp32
template <class C, bool TWO = false>
__device__ __forceinline__ void seq_reduce(seq_f32x16 (&acc)[C::NB], const char* tile, int sub, int dh, const seq_f32x16& w) {
  const int lane = threadIdx.x & 63;
  if constexpr (C::ES == 2) {
    const int g = lane >> 4, i = lane & 15, h = g >> 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      seq_bf16x8 b[TWO ? 2 : C::PL];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (C::PL == 3) {
          __bf16 x, y, z;
          seq_split3(w[8 * t + j], x, y, z);
          b[0][j] = x; b[1][j] = y; b[2][j] = z;
        } else {
          b[0][j] = (__bf16)w[8 * t + j];
          if constexpr (TWO) b[1][j] = (__bf16)(w[8 * t + j] - (float)b[0][j]);
        }
      }
      const int row0 = 32 * sub + 16 * t + 4 * h + (i >> 2), row1 = row0 + 8;
      const int col = 2 * (dh * C::DH + 16 * (g & 1)) + 8 * (i & 3);                // byte within the row, block 0
      const int x0 = seq_swz<C>(row0) << 4, x1 = seq_swz<C>(row1) << 4;
#pragma unroll
      for (int nb = 0; nb < C::NB; ++nb) {
        seq_u32x4 a[C::PL];
#pragma unroll
        for (int pl = 0; pl < C::PL; ++pl) {
          typedef __attribute__((address_space(3))) seq_s16x4 lds_s16x4;
          const char* p = tile + pl * C::kPlaneBytes;
          const seq_s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + row0 * C::RS + ((col + 64 * nb) ^ x0)));
          const seq_s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + row1 * C::RS + ((col + 64 * nb) ^ x1)));
          typedef short s16x8 __attribute__((ext_vector_type(8)));
          a[pl] = __builtin_bit_cast(seq_u32x4, s16x8{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]});
        }
        if constexpr (C::PL == 3)
          acc[nb] = seq_six(acc[nb], a[0], a[1], a[2], __builtin_bit_cast(seq_u32x4, b[0]), __builtin_bit_cast(seq_u32x4, b[1]),
                            __builtin_bit_cast(seq_u32x4, b[2]));
        else
          acc[nb] = seq_mma(acc[nb], a[0], __builtin_bit_cast(seq_u32x4, b[0]));
        if constexpr (TWO) acc[nb] = seq_mma(acc[nb], a[0], __builtin_bit_cast(seq_u32x4, b[1]));
      }
    }
  } else {
    const int m = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = 32 * sub + 8 * (i >> 2) + 4 * h + (i & 3);
      const int col = 4 * (dh * C::DH + m), x = seq_swz<C>(row) << 4;
#pragma unroll
      for (int nb = 0; nb < C::NB; ++nb) {
        const float a = *reinterpret_cast<const float*>(tile + row * C::RS + ((col + 128 * nb) ^ x));
        acc[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w[i], acc[nb], 0, 0, 0);
      }
    }
  }
}

// Own rows (bits of the answer) whose sums are not finite.  A matrix instruction multiplies what a mask hides by an exact 0,
// which is right unless that row holds an infinity or NaN (0 * inf): such own rows are done again, pair by pair over the
// visible rows alone, so that what a mask hides cannot spread.  The waves of a team share the answer.
// Every wave of the workgroup calls this (barriers inside).
template <class C>
__device__ __forceinline__ uint32_t seq_bad_rows(const seq_f32x16 (&acc)[C::NB], uint32_t more, int* red) {
  bool bad = false;
#pragma unroll
  for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
    for (int e = 0; e < 16; ++e) bad |= !(fabsf(acc[nb][e]) < INFINITY);
  const uint64_t b = __ballot(bad);
  uint32_t rows = (uint32_t)b | (uint32_t)(b >> 32) | more;
  if constexpr (C::DS > 1) {
    const int w = threadIdx.x >> 6, first = w - w % C::DS;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[w] = (int)rows;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < C::DS; ++m) rows |= (uint32_t)red[first + m];
  }
  return __builtin_amdgcn_readfirstlane(rows);
}

// one row spread over a wave: lane holds columns lane, lane + 64, ...
struct SeqSpread { float x[4]; };
template <class T>
__device__ __forceinline__ SeqSpread seq_spread(const char* p, int d) {
  SeqSpread r;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < 4; ++u) r.x[u] = lane + 64 * u < d ? SeqElt<T>::at(p + (int64_t)(lane + 64 * u) * sizeof(T)) : 0.f;
  return r;
}
__device__ __forceinline__ float seq_spread_dot(const SeqSpread& a, const SeqSpread& b) {
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < 4; ++u) s = fmaf(a.x[u], b.x[u], s);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
  return s;
}
template <class T>
__device__ __forceinline__ void seq_spread_store(char* out, char* out_lo, const float (&x)[4], float mul, int d) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (lane + 64 * u >= d) continue;
    const float y = x[u] * mul;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float*>(out)[lane + 64 * u] = y;
    } else {
      const float z = SeqElt<T>::round(y);
      reinterpret_cast<uint16_t*>(out)[lane + 64 * u] = (uint16_t)SeqElt<T>::bits(z);
      if (out_lo) reinterpret_cast<uint16_t*>(out_lo)[lane + 64 * u] = (uint16_t)SeqElt<T>::bits(y - z);
    }
  }
}

// ---- partial score blocks of the DS waves (a team) that share own rows.  A wave stores its block as four quads (registers
// 4g .. 4g + 3), a quad as 16 bytes a lane; the barrier between writing and reading is the caller's.
__device__ __forceinline__ seq_f32x4 seq_quad(const seq_f32x16& s, int g) {
  return seq_f32x4{s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]};
}
__device__ __forceinline__ void seq_set_quad(seq_f32x16& s, int g, seq_f32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s[4 * g + i] = x[i];
}
__device__ __forceinline__ seq_f32x4* seq_slot(char* at, int slot) {
  return reinterpret_cast<seq_f32x4*>(at + slot * 1024) + (threadIdx.x & 63);
}
// B blocks a wave.  Member j of a team finishes quads j * GP .. (j + 1) * GP - 1: everyone puts the quads that are not its own;
// after a barrier the finisher adds up its quads and leaves what it made of a quad in a slot of it that nobody but itself has read;
// after another barrier take() has the whole blocks.
template <class C, int B>
struct SeqShare {
  static constexpr int GP = 4 / C::DS, kSlots = 4 - GP, kWave = B * kSlots * 1024;
  static __device__ __forceinline__ seq_f32x4* slot(char* xch, int first, int j, int block, int g) {     // of quad g in member j's area
    return seq_slot(xch, ((first + j) * B + block) * kSlots + (g < j * GP ? g : g - GP));
  }
  static __device__ __forceinline__ void put(const seq_f32x16& s, char* xch, int first, int j, int block) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (g / GP != j) *slot(xch, first, j, block, g) = seq_quad(s, g);
  }
  // own quad i (number j * GP + i) over all members, one after the other from the next one on
  static __device__ __forceinline__ seq_f32x4 sum(const seq_f32x16& s, char* xch, int first, int j, int block, int i) {
    seq_f32x4 r = seq_quad(s, i);
#pragma unroll
    for (int o = 1; o < C::DS; ++o) {
      const seq_f32x4 q = seq_quad(s, o * GP + i);
#pragma unroll
      for (int u = 0; u < 4; ++u) r[u] = j == o ? q[u] : r[u];
    }
#pragma unroll
    for (int o = 1; o < C::DS; ++o) r += *slot(xch, first, (j + o) % C::DS, block, j * GP + i);
    return r;
  }
  static __device__ __forceinline__ void leave(seq_f32x4 x, char* xch, int first, int j, int block, int i) {
    *slot(xch, first, (j + 1) % C::DS, block, j * GP + i) = x;
  }
  static __device__ __forceinline__ void take(seq_f32x16& s, char* xch, int first, int block) {
#pragma unroll
    for (int g = 0; g < 4; ++g) seq_set_quad(s, g, *slot(xch, first, (g / GP + 1) % C::DS, block, g));
  }
};

// Z[d][own row] registers -> a contiguous output row
template <class C>
__device__ __forceinline__ void seq_store_own(const seq_f32x16 (&acc)[C::NB], float mul, char* out, char* out_lo, int dh, int d, int aln) {
  using T = typename C::E;
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = dh * C::DH + 32 * nb + 8 * q + 4 * h;
      if (col >= d) continue;
      if constexpr (C::OS == 4) {
        seq_u32x4 r;
#pragma unroll
        for (int u = 0; u < 4; ++u) r[u] = __float_as_uint(acc[nb][4 * q + u] * mul);
        seq_store16(out + 4 * col, r, 4 * (d - col), aln);
      } else {
        uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float x = acc[nb][4 * q + u] * mul, y = SeqElt<T>::round(x);
          hi[u >> 1] |= SeqElt<T>::bits(y) << (16 * (u & 1));
          if (out_lo) lo[u >> 1] |= SeqElt<T>::bits(x - y) << (16 * (u & 1));
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          char* o = k ? out_lo : out;
          const uint32_t* v = k ? lo : hi;
          if (!o) continue;
          if (col + 4 <= d && aln >= 8) {
            *reinterpret_cast<uint2*>(o + 2 * col) = make_uint2(v[0], v[1]);
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (col + u < d) *reinterpret_cast<uint16_t*>(o + 2 * (col + u)) = (uint16_t)(v[u >> 1] >> (16 * (u & 1)));
          }
        }
      }
    }
}

// ... -> a row of fp32 partial sums
template <class C>
__device__ __forceinline__ void seq_store_part(const seq_f32x16 (&acc)[C::NB], float mul, float* out, int dh, int d, int aln) {
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int nb = 0; nb < C::NB; ++nb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = dh * C::DH + 32 * nb + 8 * q + 4 * h;
      if (col >= d) continue;
      seq_u32x4 r;
#pragma unroll
      for (int u = 0; u < 4; ++u) r[u] = __float_as_uint(acc[nb][4 * q + u] * mul);
      seq_store16(reinterpret_cast<char*>(out + col), r, 4 * (d - col), aln);
    }
}

// ---- score arithmetic: z in base-2 units (z * log2 e), so that exp is one v_exp_f32 --------------------------------------
// z = cap * tanh(scale * s / cap) - slope * |base - key|; without a cap z = scale * s - slope * |base - key|
struct SeqScore {
  float mul, capl, slope;                 // scale*log2e (or scale / cap), cap*log2e, slope*log2e
  __device__ __forceinline__ SeqScore(const SeqAttnArgs& A, int head)
      : mul(A.cap > 0.f ? A.scale / A.cap : A.scale * kSeqLog2e), capl(A.cap * kSeqLog2e), slope(A.slope ? A.slope[head] * kSeqLog2e : 0.f) {}
};
// How a kernel bends its scores: not at all, by tanh with an absolute error of some 2^-23 (kSeqCapNear), or with a relative one (kSeqCap).
// bfloat16 takes the first of the two up to a cap of kSeqNearCap, where what it is off by, times the cap, is 2e-4 of a probability at
// most (256 scores of unit variance: 5e-5 in the 2-norm), against 2^-8 = 4e-3 for the result's own rounding.  Beyond, it would take
// the scores with it -- 4e-4 at a cap of 1e4, 5 % at 1e6, one value for all of them at 1e9 -- and float32 has no such room.
constexpr int kSeqCapNone = 0, kSeqCapNear = 1, kSeqCap = 2;
constexpr float kSeqNearCap = 1024.f;
// Without branches.  NEAR: 1 - 2 / (1 + e^2x), absolute error about 1.2e-7.  Else that form from |x| = 0.55 on (where it is good to
// 3 * 2^-24 of itself), below it the Taylor series up to x^15 (its next term is under 2^-24 of x there)
template <bool NEAR>
__device__ __forceinline__ float seq_tanh(float x) {
  const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f((NEAR ? x : fabsf(x)) * (2.f * kSeqLog2e)));
  if constexpr (NEAR) return big;
  const float y = x * x;
  float p = -929569.f / 638512875.f;
  p = fmaf(p, y, 21844.f / 6081075.f);
  p = fmaf(p, y, -1382.f / 155925.f);
  p = fmaf(p, y, 62.f / 2835.f);
  p = fmaf(p, y, -17.f / 315.f);
  p = fmaf(p, y, 2.f / 15.f);
  p = fmaf(p, y, -1.f / 3.f);
  const float small = fmaf(p * y, x, x);
  return fabsf(x) < 0.55f ? small : copysignf(big, x);
}
// one pair's z from its scaled-less product; slope_z = dz / d(scale * product) where a cap bends it
__device__ __forceinline__ float seq_z(const SeqAttnArgs& A, const SeqScore& sc, float s, int base, int key, float& slope_z) {
  slope_z = 1.f;
  if (A.cap > 0.f) {
    const float t = seq_tanh<false>(s * sc.mul);
    slope_z = 1.f - t * t;
    s = sc.capl * t;
  } else {
    s *= sc.mul;
  }
  return A.slope ? fmaf(-sc.slope, fabsf((float)(base - key)), s) : s;
}

// whether sequences have fewer than n rows on average, of queries or of keys
inline bool seq_fewer_rows(const SeqAttnArgs& A, int64_t n) { return (A.tq < A.tk ? A.tq : A.tk) < n * A.nseq; }

// workgroups of one head's neighbouring tiles on one XCD (they share its L2): blocks are dealt to the 8 XCDs in turn
__device__ __forceinline__ int seq_xcd_order(int b, int n) {
  const int q = n >> 3, r = n & 7, x = b & 7, i = b >> 3;
  return x < r ? x * (q + 1) + i : r * (q + 1) + (x - r) * q + i;
}
// Which of a head's `tiles` comes `at`-th: 8 / gcd(heads, 8) XCDs share a head, and a run of its tiles falls to each.  Where the order
// masks, the tiles' work falls (or grows) along a sequence: a run takes every n-th of them where sequences are long (a training step,
// bfloat16, 128 columns: 16384 rows, 2 heads 1247 -> 1146 us; 2 x 8192, 8 heads over 2, 1559 -> 1539), neighbours where they are short
// (96 of 37 .. 500 rows, 8 over 2, 64 columns: 286 us, spread 293).
__device__ __forceinline__ int seq_spread_tile(const SeqAttnArgs& A, int at, int tiles, int heads) {
  const int n = A.causal && A.tk >= 1024 * (int64_t)A.nseq ? 8 / min(heads & -heads, 8) : 1, q = tiles / n, r = tiles - q * n;
  const bool longer = at < r * (q + 1);
  const int run = longer ? at / (q + 1) : r + (at - r * (q + 1)) / max(q, 1);
  return (longer ? at - run * (q + 1) : at - r - run * q) * n + run;
}

}  // namespace sttran
