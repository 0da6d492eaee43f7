// Tiles of a paged cache's rows as operands of the matrix instructions, shared by the kernels that attend them
// (gfx950).
#pragma once

#include <type_traits>

#include "dsqg_mfma.hpp"
#include "dsqg_paged.hpp"

namespace dsqg {

constexpr int kWaves = kBlock / 64;
constexpr int kTile = 32;  // rows of a wave's tile: two 16-row halves

template <bool F16>
__device__ __forceinline__ f32x4_t mfma32(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return mfma_16x16x32(as_bf16x8(a), as_bf16x8(b), c);
}

// Eight stored elements as 16-bit operand values (codes of 8-bit types become bf16, exactly).
template <int CT>
__device__ __forceinline__ uint4 operand(const Raw8<CT>& r) {
  if constexpr (!narrow(CT)) {
    return r.a;
  } else if constexpr (CT == DSQG_E4M3) {
    auto cvt = [](uint32_t w, auto hi) {
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, decltype(hi)::value));
    };
    return make_uint4(cvt(r.a.x, std::false_type{}), cvt(r.a.x, std::true_type{}), cvt(r.a.y, std::false_type{}),
                      cvt(r.a.y, std::true_type{}));
  } else {
    float x[8];
    raw_floats<CT>(r, x);
    return make_uint4(cvt_pk_bf16(x[0], x[1]), cvt_pk_bf16(x[2], x[3]), cvt_pk_bf16(x[4], x[5]), cvt_pk_bf16(x[6], x[7]));
  }
}

// Eight floats as two bf16 terms: x = hi + lo exactly for a float16 value, to 2^-17 x otherwise.
__device__ __forceinline__ void split8(const float (&x)[8], uint4& hi, uint4& lo) {
  s16x4_t h0, l0, h1, l1;
  split_bf16x4(x[0], x[1], x[2], x[3], h0, l0);
  split_bf16x4(x[4], x[5], x[6], x[7], h1, l1);
  const uint2 a = __builtin_bit_cast(uint2, h0), b = __builtin_bit_cast(uint2, h1);
  const uint2 c = __builtin_bit_cast(uint2, l0), d = __builtin_bit_cast(uint2, l1);
  hi = make_uint4(a.x, a.y, b.x, b.y);
  lo = make_uint4(c.x, c.y, d.x, d.y);
}

// Eight weights (none negative) as two 16-bit terms, hi rounded down and lo what remains, so that neither is
// negative.  Where values may be infinite (INF: not in 8 bits) both terms of a weight above zero are above zero,
// for an infinity times both is that infinity, but times zero NaN.  In bf16 hi is, and lo is 2^-126 at least; in
// float16, whose smallest number is 2^-24, both are that at least (so that a weight is up to 2^-23 too large).
template <bool F16, bool INF>
__device__ __forceinline__ void split_weights(const float (&w)[8], uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = w[2 * i], b = w[2 * i + 1];
    if constexpr (F16) {
      const float s = fminf(a * 0x1p126f, 0x1p-24f), t = fminf(b * 0x1p126f, 0x1p-24f);  // 0 for 0
      h[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a + s, b + t));
      const f16x2_t q = __builtin_bit_cast(f16x2_t, h[i]);
      l[i] = __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)fmaxf(a - (float)q[0], s), (_Float16)fmaxf(b - (float)q[1], t)});
    } else {
      h[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);  // the upper halves
      float x = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), y = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
      if constexpr (INF) {
        x = fmaxf(x, fminf(a, 0x1p-126f));
        y = fmaxf(y, fminf(b, 0x1p-126f));
      }
      l[i] = cvt_pk_bf16(x, y);
    }
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// Where the contraction's steps lie in a row.  A step is 32 elements, eight for each g.  16-bit rows: elements
// 32 s + 8 g.  8-bit rows: pairs of steps of 64 elements, 64 p + 16 g + 8 (s % 2), so that a lane's
// sixteen are one piece, and what is left (D % 64) 8 g behind them.
template <int CT, int D>
struct Steps {
  static constexpr int count = Geo<D>::KS;
  static constexpr int pairs = narrow(CT) ? D / 64 : 0;
  static __device__ __forceinline__ int at(int s, int g) {
    return s < 2 * pairs ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 64 * pairs + 32 * (s - 2 * pairs) + 8 * g;
  }
};

// A tile's value rows over lanes, in pieces of 16 bytes: VL lanes a row, VP pieces a lane.
template <int CT, int D>
struct ValueMap {
  static constexpr int pieces = D * elem_size(CT) / 16;
  static constexpr int lanes = pieces == 24                                  ? 8
                               : pieces == 10 || pieces == 12 || pieces == 20 ? 4
                               : pieces == 5 || pieces == 6                   ? 2
                                                                              : pieces;
  static constexpr int per_lane = (pieces + lanes - 1) / lanes;
  static constexpr int rows = 64 / lanes;
  static constexpr int passes = kTile / rows;
};

}  // namespace dsqg
