// Attention within a window and its sinks: tiles, operands and masks shared by the forward and backward kernels (gfx950).
//
//   position i sees position j:  j <= i  and  (i - j < window  or  j < sinks),   i < length of the sequence
//
// All products are 32 x 32 tiles of the matrix instructions: v_mfma_f32_32x32x16 of 16-bit operands, v_mfma_f32_32x32x2 of
// float32 ones.  A wave owns 32 columns (queries; in dk/dv keys) whose operands stay in registers, and streams rows
// through LDS.  With rows x columns products S = A B the result lies so that a lane has sixteen rows of its column, and
// those sixteen, packed, are at once the B operand of the product that contracts over rows (weights times values, and
// so on): lane (c, h), c = l % 32, h = l / 32, register r holds row 2 E (r / E) + E h + r % E, E elements a fragment
// (8 of 16 bits, 4 of 32).  For 16 bits the A operand's rows are read in an order that makes it so: the instruction
// gives register r the row 8 (r / 4) + 4 h + r % 4, so row m of the operand is the tile's row with bits 2 and 3 of m exchanged.
//
// Rows come in with buffer loads whose resource ends at the sequence's length: what lies behind reads as zeros.
#pragma once

#include <type_traits>

#include "../../include/dsqg.h"
#include "dsqg_launch.hpp"
#include "dsqg_mfma.hpp"

namespace dsqg {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

struct WindowRows {  // rows [B, H, N, D]: base and strides in bytes
  char* at;
  long long b, h, n;
};

struct WindowParams {
  int B, Hkv, G, N, D;
  int window, sinks;
  float scale, scale2;         // softmax_scale, and times log2(e)
  const long long* lengths;    // or null: N
  WindowRows q, k, v, out, dout, dq, dk, dv;
  WindowRows low;              // what out's rounding took off (low_part), or null
  float2* stats;               // [B, H, N]: the weights' reference exponent and 1 / sum (forward: or null)
  float* delta;                // [B, H, N]: dout . out
  int waves, blocks;           // waves of a workgroup, 32 queries each; query blocks of a head
  // dk/dv: keys of a block, and blocks; those below `split` hold sinks whose far queries are other workgroups': `far` of
  // them for each.
  int kcols, kblocks, split, far;
  float* part;                 // [B, Hkv, split, 1 + far, 2, kcols, D]
};

// Whether a query workgroup may have eight waves rather than four: the rows' loads and stores to LDS are shared by twice the
// queries, the barriers by twice the waves.  Rows of 16 bits above 64 elements gain (D = 128 at B1 H16 Hkv4 N16384 window 1024:
// dq 364 us to 426, forward 262 to 268), shorter ones lose (D = 32 at B8 H8 N2048 window 256: 39.5 to 35.2 and 39.1 to 32.5).
constexpr bool may_be_wide(int T, int D) { return T != DSQG_F32 && D > 64; }

// Pairs of waves of a dk/dv workgroup, of 32 keys each: four, whose tiles and operands fit LDS but at 128 elements of float32.
constexpr int key_pairs(int T, int D) { return T == DSQG_F32 && D > 96 ? 2 : 4; }

__device__ __forceinline__ int window_length(const WindowParams& p, int b) {
  return p.lengths ? (int)max(0ll, min((long long)p.N, p.lengths[b])) : p.N;
}

template <int T> struct Op;  // T: DSQG_F32, DSQG_BF16, DSQG_F16
template <> struct Op<DSQG_F32> { static constexpr int size = 4, E = 4; typedef float elem; };
template <> struct Op<DSQG_BF16> { static constexpr int size = 2, E = 8; typedef bf16_t elem; };
template <> struct Op<DSQG_F16> { static constexpr int size = 2, E = 8; typedef bf16_t elem; };

// A fragment: 16 bytes of a row.
template <int T>
__device__ __forceinline__ f32x16_t mma(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (T == DSQG_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
  } else if constexpr (T == DSQG_BF16) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  }
  return c;
}

__device__ __forceinline__ f32x16_t zero_tile() {
  f32x16_t z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// A tile's rows in LDS.  16 bits: 16-byte pieces in rows of a power of two of them, piece i of row r in slot i ^ f(r), so that
// neither reads of one piece of sixteen rows (row_frag) nor of four pieces of four rows (col_frag) meet in a bank: with rows
// padded by a piece instead the latter took four times their cycles, half of all of LDS's.  float32, which the matrix
// instructions bound by far: rows padded by a piece.
template <int T, int D>
struct Tile {
  using O = Op<T>;
  static constexpr int E = O::E;
  static constexpr int SLOTS = D <= 32 ? 4 : D <= 64 ? 8 : 16;
  static constexpr int RB = T == DSQG_F32 ? (D + E) * 4 : SLOTS * 16;  // bytes of a row
  static constexpr int KS = D / (2 * E);         // fragments of a row
  static constexpr int DB = (D + 31) / 32;       // 32-wide blocks of a row
  static constexpr int C = 16 / E;               // fragments of a block of 32 rows as an operand
  static constexpr int PPR = D * O::size / 16;   // 16-byte pieces of a row
  // Bytes of `rows` staged rows (float32: the reads of the last block may run past a row of D = 80).
  static constexpr int bytes(int rows) { return rows * RB + (T == DSQG_F32 && D % 32 ? 64 : 0); }
  // Which slots a row's pieces are in: f(row).
  static __device__ __forceinline__ int flip(int row) {
    if constexpr (T == DSQG_F32) return 0;
    else if constexpr (SLOTS == 4) return (row >> 2) & 3;
    else if constexpr (SLOTS == 8) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return ((row & 3) << 2) | ((row >> 2) & 3);
  }
};

template <int T, int D> using Acc = f32x16_t[Tile<T, D>::DB];  // a wave's [D x 32] sums
template <int T> using Weights = u32x4_t[16 / Op<T>::E];      // 32 x 32 values as an operand

// Row l % 32 of the A operand as the tile's row (see above).
template <int T>
__device__ __forceinline__ int operand_row(int l) {
  const int m = l & 31;
  if constexpr (T == DSQG_F32) return m;
  else return (m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1);
}

// Fragment s of the A operand whose rows, 32 from a multiple of 32 on, begin at `rows` (LDS).
template <int T, int D>
__device__ __forceinline__ u32x4_t row_frag(const char* rows, int l, int s) {
  using X = Tile<T, D>;
  const int row = operand_row<T>(l);
  return *reinterpret_cast<const u32x4_t*>(rows + row * X::RB + ((2 * s) ^ ((l >> 5) ^ X::flip(row))) * 16);
}

// Fragment c of the A operand whose rows are the elements 32 d + l % 32 and whose contraction runs over those rows.
template <int T, int D>
__device__ __forceinline__ u32x4_t col_frag(const char* rows, int l, int c, int d) {
  using X = Tile<T, D>;
  if constexpr (T == DSQG_F32) {
    const float* t = reinterpret_cast<const float*>(rows + (8 * c + 4 * (l >> 5)) * X::RB) + 32 * d + (l & 31);
    u32x4_t f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __float_as_uint(t[e * (X::RB / 4)]);
    return f;
  } else {
    const int row = 8 * (l >> 5) + ((l & 15) >> 2), piece = ((l & 16) >> 3) | ((l & 3) >> 1);
    auto at = [&](int q) {
      return reinterpret_cast<const bf16_t*>(rows + (row + 4 * q) * X::RB + ((4 * d) ^ (piece ^ X::flip(row + 4 * q))) * 16 + 8 * (l & 1) +
                                             16 * c * X::RB);
    };
    const uint2 a = __builtin_bit_cast(uint2, lds_read_tr16(at(0))), b = __builtin_bit_cast(uint2, lds_read_tr16(at(1)));
    return u32x4_t{a.x, a.y, b.x, b.y};
  }
}

// Sixteen values of a column as the B operand that contracts over the tile's rows.  16-bit values are rounded once.
template <int T>
__device__ __forceinline__ void pack(const float (&w)[16], Weights<T>& f) {
  if constexpr (T == DSQG_F32) {
#pragma unroll
    for (int r = 0; r < 16; ++r) f[r / 4][r % 4] = __float_as_uint(w[r]);
  } else {
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      if constexpr (T == DSQG_BF16) f[r / 8][r % 8 / 2] = cvt_pk_bf16(w[r], w[r + 1]);
      else f[r / 8][r % 8 / 2] = __builtin_bit_cast(uint32_t, half2_t{(_Float16)w[r], (_Float16)w[r + 1]});
    }
  }
}

// The tile's row of register r.
template <int T>
__device__ __forceinline__ constexpr int reg_row(int r, int h) {
  constexpr int E = Op<T>::E;
  return 2 * E * (r / E) + E * h + r % E;
}

// Rows of a tile on their way from memory to LDS: every one of the workgroup's NT threads has the same pieces of each tile.
template <int T, int D, int RT, int NT = kBlock>
struct Stage {
  using X = Tile<T, D>;
  static constexpr int U = (RT * X::PPR + NT - 1) / NT;
  u32x4_t x[U];
  // Rows `row0` on of a head's rows; those from `length` on are zeros.  (Row strides are below 2^24 bytes.)
  __device__ __forceinline__ void load(const char* head, long long stride, int row0, int length) {
    const int n = min(RT, length - row0);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(head) + row0 * stride, (short)0,
                                                                       n > 0 ? (n - 1) * (int)stride + D * X::O::size : 0, 0x00020000);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = threadIdx.x + u * NT, row = e / X::PPR;
      x[u] = __builtin_amdgcn_raw_buffer_load_b128(r, row * (int)stride + (e - row * X::PPR) * 16, 0, 0);
    }
  }
  __device__ __forceinline__ void store(char* rows) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = threadIdx.x + u * NT, row = e / X::PPR;
      if (RT * X::PPR % NT == 0 || row < RT)
        *reinterpret_cast<u32x4_t*>(rows + row * X::RB + ((e - row * X::PPR) ^ X::flip(row)) * 16) = x[u];
    }
  }
  // Times 2^-30.
  __device__ __forceinline__ void shrink() {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = x[u][e];
        if constexpr (T == DSQG_F32)
          x[u][e] = __float_as_uint(__uint_as_float(w) * 0x1p-30f);
        else
          x[u][e] = (__float_as_uint(__uint_as_float(w & 0xffff0000u) * 0x1p-30f) & 0xffff0000u) |
                    (__float_as_uint(__uint_as_float(w << 16) * 0x1p-30f) >> 16);
      }
    }
  }
  // Puts zeros in the place of infinities and NaN, which times the weight of a column that does not see them would be no
  // zero (add_odd); says whether this thread's pieces held any.
  __device__ __forceinline__ bool clean() {
    constexpr uint32_t m = T == DSQG_F32 ? 0x7f800000u : T == DSQG_BF16 ? 0x7f80u : 0x7c00u;
    uint32_t odd = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t gone = (x[u][e] & m) == m ? 0xffffu : 0u;
        if constexpr (T == DSQG_F32) gone |= gone << 16;
        else gone |= (x[u][e] & (m << 16)) == m << 16 ? 0xffff0000u : 0u;
        x[u][e] &= ~gone;
        odd |= gone;
      }
    }
    return odd != 0;
  }
};

// acc[d] += A^T w over the 32 rows at `rows`: each block's fragments are on their way while the one before is multiplied.
template <int T, int D>
__device__ __forceinline__ void contract(Acc<T, D>& acc, const char* rows, int l, const Weights<T>& w) {
  using X = Tile<T, D>;
  u32x4_t f[2][X::C];
#pragma unroll
  for (int c = 0; c < X::C; ++c) f[0][c] = col_frag<T, D>(rows, l, c, 0);
#pragma unroll
  for (int d = 0; d < X::DB; ++d) {
    if (d + 1 < X::DB) {
#pragma unroll
      for (int c = 0; c < X::C; ++c) f[(d + 1) & 1][c] = col_frag<T, D>(rows, l, c, d + 1);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < X::C; ++c) acc[d] = mma<T>(f[d & 1][c], w[c], acc[d]);
  }
}

// The scores of the 32 rows at `rows` with the columns in b.
template <int T, int D>
__device__ __forceinline__ f32x16_t scores(const char* rows, int l, const u32x4_t (&b)[Tile<T, D>::KS]) {
  using X = Tile<T, D>;
  constexpr int AHEAD = T == DSQG_F32 ? 4 : X::KS;  // (all of a row's fragments, 32 registers at most, before the first product)
  u32x4_t a[AHEAD];
#pragma unroll
  for (int e = 0; e < AHEAD; ++e) a[e] = row_frag<T, D>(rows, l, e);
  __builtin_amdgcn_sched_barrier(0);
  f32x16_t s = zero_tile();
#pragma unroll
  for (int e = 0; e < X::KS; ++e) {
    s = mma<T>(a[e % AHEAD], b[e], s);
    if (e + AHEAD < X::KS) a[e % AHEAD] = row_frag<T, D>(rows, l, e + AHEAD);
  }
  return s;
}

// The same of rows as they are in memory, of which `have` exist: those of a tile that Stage::clean took something out of.
template <int T, int D>
__device__ __forceinline__ f32x16_t scores_as_stored(const char* rows, long long stride, int have, int l, const u32x4_t (&b)[Tile<T, D>::KS]) {
  using X = Tile<T, D>;
  asm volatile("");  // (a branch)
  const int row = operand_row<T>(l);
  f32x16_t s = zero_tile();
#pragma unroll
  for (int e = 0; e < X::KS; ++e) {
    u32x4_t a = {0u, 0u, 0u, 0u};
    if (row < have) a = *reinterpret_cast<const u32x4_t*>(rows + row * stride + (2 * e + (l >> 5)) * 16);
    s = mma<T>(a, b[e], s);
    __builtin_amdgcn_sched_barrier(0);
  }
  return s;
}

// Adds what Stage::clean left out of 32 rows, where the lane's column sees it: the rows as they are in memory, of which
// `have` exist.  A weight above zero times an infinity is that infinity, whatever the weight; where weights have signs, or
// the value is NaN, the sum is no number either way.  sees(row).
template <int T, int D, typename F>
__device__ __forceinline__ void add_odd(Acc<T, D>& acc, const char* rows, long long stride, int have, int l, F&& sees) {
  using X = Tile<T, D>;
  constexpr uint32_t m = T == DSQG_F32 ? 0x7f800000u : T == DSQG_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll 1
  for (int row = 0; row < min(32, have); ++row) {
    const uint32_t seen = sees(row) ? ~0u : 0u;
    const char* const from = rows + row * stride;
#pragma unroll
    for (int d = 0; d < X::DB; ++d) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = 32 * d + 8 * (r / 4) + 4 * (l >> 5) + r % 4;
        if (D % 32 != 0 && at >= D) continue;
        uint32_t x;
        if constexpr (T == DSQG_F32) x = reinterpret_cast<const uint32_t*>(from)[at];
        else x = reinterpret_cast<const bf16_t*>(from)[at];
        x &= (x & m) == m ? seen : 0u;
        if constexpr (T == DSQG_F32) acc[d][r] += __uint_as_float(x);
        else if constexpr (T == DSQG_BF16) acc[d][r] += __uint_as_float(x << 16);
        else acc[d][r] += (float)__builtin_bit_cast(_Float16, (bf16_t)x);
        if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// Exponents of weights, s c - m.  One multiply-add leaves the rounding of m, up to half its last bit: nothing while |m| is
// below kLarge (2^-8 of the weights, the same in their sum), an exponent without bounds for huge scores.  Those are rounded
// before m, the rounded largest of them, is taken from them.
constexpr float kLarge = 65536.f;

__device__ __forceinline__ float large_exponent(float s, float c, float m) {
#pragma clang fp contract(off)
  return s * c - m;
}

// The reference exponent of a largest score s, whose weight becomes 2^lift.  The score is rounded first, as large_exponent
// rounds it (in one multiply-add a huge product could end a step below the rounded score, and its weight be 2^128), and float16's
// lift is left out where that step is so large that less than 2^16 of it could become more: its largest weight is 1 there.
template <int T>
__device__ __forceinline__ float reference_exponent(float s, float c, float lift) {
#pragma clang fp contract(off)
  const float m = s * c;
  return T == DSQG_F16 && fabsf(m) >= kLarge ? m : m - lift;
}

// s to exponents; m(r) of each value.
template <typename F>
__device__ __forceinline__ void exponents(float (&s)[16], float c, bool large, F&& m) {
  if (__builtin_expect(large, 0)) {
    asm volatile("");  // (a branch: as a choice it costs three more instructions for each value)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = large_exponent(s[r], c, m(r));
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], c, -m(r));
  }
}

// Which of a tile's 32 rows a column sees: those `lo` .. `hi`, and the first `sinks`.  (Bounds in 32 bits: positions and
// windows are 2^30 at most.)
struct Seen {
  int lo, hi, sinks;
  __device__ __forceinline__ bool operator()(int row) const { return row <= hi && (row >= lo || row < sinks); }
};

// Puts x in the place of the values of rows that the column does not see.  Most tiles hold no sinks: one comparison then.
template <int T, int N>
__device__ __forceinline__ void hide(float x, const Seen& seen, bool sinks, int h, float (&a)[16], float (&b)[N]) {
  auto put = [&](int r, bool see) {
    a[r] = see ? a[r] : x;
    if constexpr (N == 16) b[r] = see ? b[r] : x;
  };
  if (sinks) {
#pragma unroll
    for (int r = 0; r < 16; ++r) put(r, seen(reg_row<T>(r, h)));
  } else {
    const unsigned n = (unsigned)max(0, seen.hi - max(seen.lo, -64) + 1);  // (no row is below -64)
    const int lo = max(seen.lo, -64) - Op<T>::E * h;
#pragma unroll
    for (int r = 0; r < 16; ++r) put(r, (unsigned)(reg_row<T>(r, 0) - lo) < n);
  }
}

// What the rounding of x to 16 bits takes off, in float16 times 2^11, which keeps it as far from the subnormal numbers as x is.
// (None where the result is no number.)
template <int T> constexpr float low_scale() { return T == DSQG_F16 ? 2048.f : 1.f; }
template <int T>
__device__ __forceinline__ float low_part(float x) {
  float low;
  if constexpr (T == DSQG_F16) low = (x - (float)(_Float16)x) * low_scale<T>();
  else low = x - __uint_as_float(cvt_pk_bf16(x, 0.f) << 16);
  return fabsf(low) < INFINITY ? low : 0.f;
}

// A wave's 32 columns [D x 32] to rows of an output, times f (of each column), through the wave's LDS block (out_block bytes);
// n rows are stored, of columns that are not live zeros.  LOW: what their rounding takes off, in their place.
template <int T, int D>
constexpr int out_block() { return 32 * (D * Op<T>::size + 16); }

template <int T, int D, bool LOW = false>
__device__ __forceinline__ void store_columns(const Acc<T, D>& acc, float f, bool live, char* block, char* out,
                                              long long stride, int n, int l) {
  using X = Tile<T, D>;
  const int c = l & 31, h = l >> 5;
#pragma unroll
  for (int d = 0; d < X::DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int at = 32 * d + 8 * g + 4 * h;
      if (D % 32 != 0 && at >= D) continue;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = live ? acc[d][4 * g + e] * f : 0.f;
        if constexpr (LOW) x[e] = low_part<T>(x[e]);
      }
      char* to = block + c * (out_block<T, D>() / 32) + at * X::O::size;
      if constexpr (T == DSQG_F32) {
        *reinterpret_cast<f32x4_t*>(to) = f32x4_t{x[0], x[1], x[2], x[3]};
      } else {
        typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
        if constexpr (T == DSQG_BF16) {
          *reinterpret_cast<u32x2_t*>(to) = u32x2_t{cvt_pk_bf16(x[0], x[1]), cvt_pk_bf16(x[2], x[3])};
        } else {
          *reinterpret_cast<u32x2_t*>(to) = u32x2_t{__builtin_bit_cast(uint32_t, half2_t{(_Float16)x[0], (_Float16)x[1]}),
                                                    __builtin_bit_cast(uint32_t, half2_t{(_Float16)x[2], (_Float16)x[3]})};
        }
      }
    }
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int u = 0; u < 32 * X::PPR / 64; ++u) {
    const int e = l + 64 * u, row = e / X::PPR, piece = e - row * X::PPR;
    if (row < n)
      __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(block + row * (out_block<T, D>() / 32) + piece * 16),
                                  reinterpret_cast<u32x4_t*>(out + row * stride + piece * 16));
  }
}

// The tiles of RT rows that a block of columns sees: `sinks` of them from the beginning, then those from `from` on.
struct WindowSpan {
  int sinks, from, n;
  __device__ __forceinline__ int tile(int t) const { return t < sinks ? t : t - sinks + from; }
};

// Keys of the queries q0 .. q1.
template <int RT>
__device__ __forceinline__ WindowSpan keys_of(const WindowParams& p, int q0, int q1) {
  const int lo = max(0, q0 - p.window + 1);
  WindowSpan s;
  s.sinks = (min(p.sinks, lo) + RT - 1) / RT;
  s.from = max(s.sinks, lo / RT);
  s.n = s.sinks + max(0, q1 / RT + 1 - s.from);
  return s;
}

hipError_t launch_window_fwd(const WindowParams& p, int dtype, hipStream_t st);
hipError_t launch_window_bwd(const WindowParams& p, int dtype, hipStream_t st);

}  // namespace dsqg
