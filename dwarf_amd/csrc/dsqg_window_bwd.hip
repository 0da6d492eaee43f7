// Attention within a window and its sinks, backward (gfx950).
//
//   p_ij = 2^(scale2 q_i.k_j - m_i) / sum_i,   D_i = dout_i . out_i,   dS_ij = p_ij (dout_i . v_j - D_i)
//
// (out as the forward summed it: its 16-bit value and what the rounding took off.  From the 16-bit value alone D_i is off by more
// than all of dS_ij where a query has nearly all its weight on one key: dq and dk by 0.0055 of their norm with a window of 2 in
// bfloat16, against 0.0023 so and the 0.0017 that the results' own rounding is.)
//
//   dq_i = scale sum_j dS_ij k_j,   dk_j = scale sum_i dS_ij q_i,   dv_j = sum_i p_ij dout_i
//
// Two launches, neither of which needs an atomic: dq with a wave's 32 queries as columns, over the tiles of keys and values
// that they see, as in the forward (it also leaves D); dk and dv with 32 keys as columns, over the tiles of queries that see
// them, those of all query heads of the key/value head one after another.  Scores and dout . v are computed in both:
// seven products where one pass over pairs would have five, but the sums stay in registers and their order is fixed.
//
// The sinks are seen by all queries behind them: a key block that holds sinks would take as long as the sequence is,
// where the others take a window.  Its queries beyond the window are split over further workgroups, and a third
// launch adds the parts.
//
// p and dS enter the products rounded to the 16-bit type (2^-8 of each in bfloat16, 2^-11 in float16, where factors keep them in
// its range); float32 operands are not rounded.  Everything else is fp32.
//
// Measured (bfloat16): B1 H16 Hkv4 N16384 D128 window 1024, dq 383 us, dk/dv 476 us, 560 TFLOP/s of the seven products; B8 H8
// Hkv8 N2048 D32 window 256 with 4 sinks, dq 32 us, dk/dv 43 us, their parts' sum 4.9 us.  Latency bounds both: vector instructions
// issue in 28 and 25 % of the cycles at D = 128, matrix instructions in 23 and 25 %, and a tile's scores, weights and products
// follow each other; at D = 32 vector instructions issue in 25 and 33 %.  float16, with its factors: 1140 us the whole step for
// bfloat16's 1050.
#include <algorithm>

#include "dsqg_window.hpp"

namespace dsqg {
namespace {

__device__ __forceinline__ u32x4_t frag_or_zero(const char* at, bool there) {
  u32x4_t x = {0u, 0u, 0u, 0u};
  if (there) x = *reinterpret_cast<const u32x4_t*>(at);
  return x;
}

// Two floats of a fragment pair's product, over its elements.
template <int T>
__device__ __forceinline__ float dot_frag(u32x4_t a, u32x4_t b, float s) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (T == DSQG_F32) {
      s = __builtin_fmaf(__uint_as_float(a[e]), __uint_as_float(b[e]), s);
    } else if constexpr (T == DSQG_BF16) {
      s = __builtin_fmaf(__uint_as_float(a[e] << 16), __uint_as_float(b[e] << 16), s);
      s = __builtin_fmaf(__uint_as_float(a[e] & 0xffff0000u), __uint_as_float(b[e] & 0xffff0000u), s);
    } else {
      const uint32_t xe = a[e], ye = b[e];  // (a bit_cast of an element itself reads the vector's first)
      const half2_t x = __builtin_bit_cast(half2_t, xe), y = __builtin_bit_cast(half2_t, ye);
      s = __builtin_fmaf((float)x[0], (float)y[0], s);
      s = __builtin_fmaf((float)x[1], (float)y[1], s);
    }
  }
  return s;
}

// float16 operands end at 65504 and lose bits below 2^-14, where loss scales and long windows bring dS past either: it is packed
// times a power of two of its column, which its largest so far chooses (2^13 to 2^15 then) as the forward's running maximum
// does, and the column's sum is taken back by it.  p, at most 1, is packed times 2^14.
constexpr float kNoFactor = 0x1p120f;  // before the first
template <int T> constexpr float weight_factor() { return T == DSQG_F16 ? 0x1p14f : 1.f; }

// The column's factor for sixteen more values a lane.
__device__ __forceinline__ float next_factor(const float (&x)[16], float c) {
  float mx = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fabsf(x[r]));
  mx = xor32_pair_max(mx);
  if (__any(mx * c > 0x1p15f)) {
    const uint32_t e = max(__float_as_uint(mx) >> 23, 27u);  // (2^-100 at least)
    const float next = __uint_as_float((267u - e) << 23);    // 2^13 over mx's power of two
    c = mx * c > 0x1p15f ? next : c;
  }
  return c;
}

// next / c of two powers of two, next the smaller.
__device__ __forceinline__ float factor_ratio(float next, float c) {
  const int e = (int)(__float_as_uint(next) >> 23) - (int)(__float_as_uint(c) >> 23) + 127;
  return e > 0 ? __uint_as_float((uint32_t)e << 23) : 0.f;
}

template <int N>
__device__ __forceinline__ void refactor(f32x16_t (&acc)[N], float& c, float next) {
  if (__any(next != c)) {
    const float f = factor_ratio(next, c);
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= f;
    c = next;
  }
}

// 1 / c, and what else a sum is multiplied by in the end.
__device__ __forceinline__ float unfactor(float c, float f) { return __uint_as_float((254u << 23) - __float_as_uint(c)) * f; }

template <int T, int D, int NW>
__global__ __launch_bounds__(64 * NW, D <= 32 ? 4 : 2) void window_dq_kernel(WindowParams p) {
  using X = Tile<T, D>;
  constexpr int RT = T == DSQG_F32 || D > 64 ? 32 : 64, KB = RT / 32, TB = X::bytes(RT), kCols = 32 * NW;
  constexpr int BYTES = 4 * TB > NW * out_block<T, D>() ? 4 * TB : NW * out_block<T, D>();
  __shared__ __align__(16) char bytes[BYTES];
  auto lds = reinterpret_cast<char(*)[2][TB]>(bytes);  // [which tile][keys, values]
  __shared__ int odd[2];  // which tile's keys hold infinities or NaN, plus one

  const int block = xcd_logical_block(blockIdx.x, gridDim.x);
  const int g = block % p.G, rest = block / p.G;
  const int at = p.blocks - 1 - rest % p.blocks, bk = rest / p.blocks;
  const int b = bk / p.Hkv, hk = bk - b * p.Hkv, head = hk * p.G + g;
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = l & 31, h = l >> 5;
  const int length = window_length(p, b);
  const int q0 = at * kCols, i0 = q0 + 32 * wave, i = i0 + c;
  const char* const kh = p.k.at + b * p.k.b + hk * p.k.h;
  const char* const vh = p.v.at + b * p.v.b + hk * p.v.h;
  const WindowSpan span = q0 < length ? keys_of<RT>(p, q0, min(q0 + kCols, length) - 1) : WindowSpan{0, 0, 0};
  const long long stat = ((long long)b * p.Hkv * p.G + head) * p.N + i;

  u32x4_t q[X::KS], dout[X::KS];
  float delta = 0.f, lost = 0.f;
  {
    const char* const rq = p.q.at + b * p.q.b + head * p.q.h + (long long)i * p.q.n;
    const char* const rd = p.dout.at + b * p.dout.b + head * p.dout.h + (long long)i * p.dout.n;
    const char* const ro = p.out.at + b * p.out.b + head * p.out.h + (long long)i * p.out.n;
    const char* const rl = p.low.at + b * p.low.b + head * p.low.h + (long long)i * p.low.n;
#pragma unroll
    for (int s = 0; s < X::KS; ++s) {
      const int e = (2 * X::E * s + X::E * h) * X::O::size;
      q[s] = frag_or_zero(rq + e, i < length);
      dout[s] = frag_or_zero(rd + e, i < length);
      delta = dot_frag<T>(dout[s], frag_or_zero(ro + e, i < length), delta);
      if (T != DSQG_F32) lost = dot_frag<T>(dout[s], frag_or_zero(rl + e, i < length && p.low.at), lost);
    }
    if (T != DSQG_F32) delta += lost * (1.f / low_scale<T>());
    delta = xor32_pair_sum(delta);
  }
  float2 st = make_float2(INFINITY, 0.f);
  if (i < length) st = p.stats[stat];
  const bool large = __any(i < length && fabsf(st.x) >= kLarge);
  if (h == 0 && i < p.N) p.delta[stat] = delta;
  if (threadIdx.x < 2) odd[threadIdx.x] = 0;

  Stage<T, D, RT, 64 * NW> sk, sv;
  auto load = [&](int t) {
    sk.load(kh, p.k.n, span.tile(t) * RT, length);
    sv.load(vh, p.v.n, span.tile(t) * RT, length);
  };
  auto edge = [&](int t) {
    const int j0 = span.tile(t) * RT;
    return j0 + RT - 1 > q0 || (q0 + kCols - 1 - j0 >= p.window && j0 + RT > p.sinks);
  };
  auto store = [&](int t) {
    if (edge(t) && sk.clean()) odd[t & 1] = t + 1;
    sk.store(lds[t & 1][0]);
    sv.store(lds[t & 1][1]);
  };

  Acc<T, D> acc;
#pragma unroll
  for (int d = 0; d < X::DB; ++d) acc[d] = zero_tile();
  float factor = T == DSQG_F16 ? kNoFactor : 1.f;

  __syncthreads();
  if (span.n > 0) {
    load(0);
    store(0);
    if (span.n > 1) load(1);
  }
  __syncthreads();
#pragma unroll 1
  for (int t = 0; t < span.n; ++t) {
    const int j0 = span.tile(t) * RT;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int k0 = j0 + 32 * kb;
      const bool none = k0 > i0 + 31 || (k0 + 32 <= i0 - p.window + 1 && k0 >= p.sinks);
      const bool all = k0 + 31 <= i0 && (i0 + 31 - k0 < p.window || k0 + 32 <= p.sinks);
      if (none) continue;
      const char* const kt = lds[t & 1][0] + 32 * kb * X::RB;
      const char* const vt = lds[t & 1][1] + 32 * kb * X::RB;
      f32x16_t s = scores<T, D>(kt, l, q);
      // (A key's infinity may be a score of -infinity: without it that would be another weight.)
      if (__builtin_expect(odd[t & 1] == t + 1, 0)) s = scores_as_stored<T, D>(kh + k0 * p.k.n, p.k.n, length - k0, l, q);
      const f32x16_t dp = scores<T, D>(vt, l, dout);
      const Seen seen = {i - p.window + 1 - k0, i - k0, p.sinks - k0};
      float w[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = s[r];
      exponents(w, p.scale2, large, [&](int) { return st.x; });
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = __builtin_amdgcn_exp2f(w[r]) * st.y * (dp[r] - delta);
      if (!all) {
        float no[1];
        hide<T>(0.f, seen, k0 < p.sinks, h, w, no);
      }
      if constexpr (T == DSQG_F16) {
        refactor(acc, factor, next_factor(w, factor));
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] *= factor;
      }
      Weights<T> f;
      pack<T>(w, f);
      contract<T, D>(acc, kt, l, f);
      if (odd[t & 1] == t + 1) add_odd<T, D>(acc, kh + k0 * p.k.n, p.k.n, length - k0, l, seen);
    }
    if (t + 1 < span.n) {
      store(t + 1);
      if (t + 2 < span.n) load(t + 2);
    }
    __syncthreads();
  }
  store_columns<T, D>(acc, unfactor(factor, p.scale), i < length, bytes + wave * out_block<T, D>(),
                      p.dq.at + b * p.dq.b + head * p.dq.h + i0 * p.dq.n, p.dq.n, p.N - i0, l);
}

// What a dk/dv workgroup takes: a key block (part 0), those of a head on one XCD, or, behind all of them, a share of the far
// queries of one that holds sinks.
struct KeyBlock {
  int bk, at, part;
  __device__ __forceinline__ explicit KeyBlock(const WindowParams& p) {
    const int heads = p.B * p.Hkv, whole = heads * p.kblocks;
    if ((int)blockIdx.x < whole) {
      const int block = xcd_logical_block(blockIdx.x, whole);
      bk = block / p.kblocks;
      at = block - bk * p.kblocks;
      part = 0;
    } else {
      const int block = blockIdx.x - whole, rest = block / heads;
      bk = block - rest * heads;
      at = rest / p.far;
      part = 1 + rest - at * p.far;
    }
  }
  // The tiles of RT queries that it goes over, of each head the same; its keys are `kc`.
  __device__ __forceinline__ void queries(const WindowParams& p, int RT, int kc, int length, int& first, int& tiles) const {
    const int k0 = at * kc;
    first = k0 / RT;
    tiles = 0;
    if (k0 >= length) return;
    const int last = (length - 1) / RT;
    const int near = (int)min((long long)last, ((long long)k0 + kc - 2 + p.window) / RT);  // of the window
    if (at >= p.split) {
      tiles = (k0 < p.sinks ? last : near) + 1 - first;
    } else if (part == 0) {
      tiles = near + 1 - first;
    } else {
      const int n = last - near, lo = (int)((long long)n * (part - 1) / p.far), hi = (int)((long long)n * part / p.far);
      first = near + 1 + lo;
      tiles = hi - lo;
    }
  }
};

// Up to `kSingle` elements a wave has the scores, weights and sums of its 32 keys to itself.  (Above, pairs: the whole backward at
// B2 H16 Hkv4 N4096 window 512, bfloat16, D = 80 236 us and 96 248, by single waves 376 and 403; D = 128 see the pairs' kernel.)
constexpr int kSingle = 64;

template <int T, int D>
__global__ __launch_bounds__(kBlock, D <= 32 && T != DSQG_F32 ? 3 : 2) void window_dkdv_kernel(WindowParams p) {
  using X = Tile<T, D>;
  constexpr int RT = T == DSQG_F32 ? 32 : 64, RB = RT / 32, TB = X::bytes(RT), KC = kBlock / 2;
  static_assert(4 * TB >= 4 * out_block<T, D>(), "the waves' output rows fit the tiles");
  __shared__ __align__(16) char lds[2][2][TB];         // [which tile][queries, dout]
  __shared__ __align__(16) float rows[2][3][RT];       // ... [reference exponent, 1 / sum, D]
  __shared__ int odd[2][3];                            // ... queries, dout hold infinities or NaN; exponents are large

  const KeyBlock block(p);
  const int bk = block.bk, at = block.at, part = block.part;
  const int b = bk / p.Hkv, hk = bk - b * p.Hkv;
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = l & 31, h = l >> 5;
  const int length = window_length(p, b);
  const int k0 = at * KC, j0 = k0 + 32 * wave, j = j0 + c;

  int first, tiles;
  block.queries(p, RT, KC, length, first, tiles);
  const int steps = tiles * p.G;

  u32x4_t k[X::KS], v[X::KS];
  {
    const char* const rk = p.k.at + b * p.k.b + hk * p.k.h + (long long)j * p.k.n;
    const char* const rv = p.v.at + b * p.v.b + hk * p.v.h + (long long)j * p.v.n;
#pragma unroll
    for (int s = 0; s < X::KS; ++s) {
      const int e = (2 * X::E * s + X::E * h) * X::O::size;
      k[s] = frag_or_zero(rk + e, j < length);
      v[s] = frag_or_zero(rv + e, j < length);
    }
  }
  if (threadIdx.x < 6) odd[threadIdx.x / 3][threadIdx.x % 3] = 0;

  Stage<T, D, RT> sq, sd;
  float2 st;
  float de;
  auto row0 = [&](int t) { return (first + t % tiles) * RT; };
  auto load = [&](int t) {
    const int head = hk * p.G + t / tiles, i0 = row0(t);
    sq.load(p.q.at + b * p.q.b + head * p.q.h, p.q.n, i0, length);
    sd.load(p.dout.at + b * p.dout.b + head * p.dout.h, p.dout.n, i0, length);
    st = make_float2(INFINITY, 0.f);
    de = 0.f;
    if (threadIdx.x < RT && i0 + (int)threadIdx.x < length) {
      const long long s = ((long long)b * p.Hkv * p.G + head) * p.N + i0 + threadIdx.x;
      st = p.stats[s];
      de = p.delta[s];
    }
  };
  auto edge = [&](int t) {
    const int i0 = row0(t);
    return i0 < k0 + KC - 1 || (i0 + RT - 1 - k0 >= p.window && k0 + KC > p.sinks);
  };
  auto store = [&](int t) {
    if (edge(t)) {
      if (sq.clean()) odd[t & 1][0] = t + 1;
      if (sd.clean()) odd[t & 1][1] = t + 1;
    }
    sq.store(lds[t & 1][0]);
    sd.store(lds[t & 1][1]);
    if (threadIdx.x < RT) {
      rows[t & 1][0][threadIdx.x] = st.x;
      rows[t & 1][1][threadIdx.x] = st.y * weight_factor<T>();
      rows[t & 1][2][threadIdx.x] = de;
      if (fabsf(st.x) >= kLarge && st.x != INFINITY) odd[t & 1][2] = t + 1;
    }
  };

  Acc<T, D> dk, dv;
#pragma unroll
  for (int d = 0; d < X::DB; ++d) dk[d] = dv[d] = zero_tile();
  float factor = T == DSQG_F16 ? kNoFactor : 1.f;

  __syncthreads();
  if (steps > 0) {
    load(0);
    store(0);
    if (steps > 1) load(1);
  }
  __syncthreads();
#pragma unroll 1
  for (int t = 0; t < steps; ++t) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int i0 = row0(t) + 32 * rb;
      const bool none = i0 + 31 < j0 || (i0 - (j0 + 31) >= p.window && j0 >= p.sinks);
      const bool all = i0 >= j0 + 31 && (i0 + 31 - j0 < p.window || j0 + 32 <= p.sinks);
      if (none) continue;
      const char* const qt = lds[t & 1][0] + 32 * rb * X::RB;
      const char* const dt = lds[t & 1][1] + 32 * rb * X::RB;
      // (Rows are queries here: a sink is seen by all from itself on.)
      const Seen seen = {j - i0, j < p.sinks ? 64 : min(64, j - i0 + p.window - 1), 0};
      const f32x16_t s = scores<T, D>(qt, l, k), dp = scores<T, D>(dt, l, v);
      const bool large = odd[t & 1][2] == t + 1;
      float w[16], x[16], m[16];
#pragma unroll
      for (int r4 = 0; r4 < 16; r4 += 4) {
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(&rows[t & 1][0][32 * rb + reg_row<T>(r4, h)]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[r4 + e] = s[r4 + e];
          m[r4 + e] = y[e];
        }
      }
      exponents(w, p.scale2, large, [&](int r) { return m[r]; });
#pragma unroll
      for (int r4 = 0; r4 < 16; r4 += 4) {
        const int row = 32 * rb + reg_row<T>(r4, h);
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(&rows[t & 1][1][row]);
        const f32x4_t d = *reinterpret_cast<const f32x4_t*>(&rows[t & 1][2][row]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[r4 + e] = __builtin_amdgcn_exp2f(w[r4 + e]) * y[e];
          x[r4 + e] = w[r4 + e] * (dp[r4 + e] - d[e]);
        }
      }
      if (!all) hide<T>(0.f, seen, false, h, w, x);
      Weights<T> f;
      pack<T>(w, f);
      contract<T, D>(dv, dt, l, f);
      if constexpr (T == DSQG_F16) {
        refactor(dk, factor, next_factor(x, factor));
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= factor;
      }
      pack<T>(x, f);
      contract<T, D>(dk, qt, l, f);
      const int head = hk * p.G + t / tiles;
      if (odd[t & 1][0] == t + 1)
        add_odd<T, D>(dk, p.q.at + b * p.q.b + head * p.q.h + i0 * p.q.n, p.q.n, length - i0, l, seen);
      if (odd[t & 1][1] == t + 1)
        add_odd<T, D>(dv, p.dout.at + b * p.dout.b + head * p.dout.h + i0 * p.dout.n, p.dout.n, length - i0, l, seen);
    }
    if (t + 1 < steps) {
      store(t + 1);
      if (t + 2 < steps) load(t + 2);
    }
    __syncthreads();
  }

  const float fk = unfactor(factor, 1.f / weight_factor<T>()), fv = 1.f / weight_factor<T>();
  if (at < p.split) {
    float* const to = p.part + ((((long long)bk * p.split + at) * (1 + p.far) + part) * 2 * KC + 32 * wave + c) * D;
#pragma unroll
    for (int d = 0; d < X::DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = 32 * d + 8 * g + 4 * h;
        if (D % 32 != 0 && e >= D) continue;
        *reinterpret_cast<f32x4_t*>(to + e) = f32x4_t{dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]} * fk;
        *reinterpret_cast<f32x4_t*>(to + KC * D + e) = f32x4_t{dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]} * fv;
      }
    return;
  }
  char* const mine = lds[0][0] + wave * out_block<T, D>();
  store_columns<T, D>(dk, fk * p.scale, j < length, mine, p.dk.at + b * p.dk.b + hk * p.dk.h + j0 * p.dk.n, p.dk.n, p.N - j0, l);
  store_columns<T, D>(dv, fv, j < length, mine, p.dv.at + b * p.dv.b + hk * p.dv.h + j0 * p.dv.n, p.dv.n, p.N - j0, l);
}

// Eight waves for 128 keys: a key's scores and weights take registers for its own key and value, its sums for two rows of
// D more, and one wave with both leaves no place for a second one on its SIMD (D = 128: 978 us at B1 H16 Hkv4 N16384 window 1024).
// So waves 0-3 make p and dS of 32 keys each, and waves 4-7, a step of 32 queries behind, multiply them with the rows: the
// operands go through LDS lane by lane, 64 bytes each way, and a SIMD has one of each kind, whose vector and matrix work overlap.
constexpr int kSteps = 3;  // tiles in LDS: one used by each kind, one arriving
template <int T, int D> constexpr int dkdv_threads() { return 2 * 64 * key_pairs(T, D); }

template <int T, int D>
__global__ __launch_bounds__((dkdv_threads<T, D>()), key_pairs(T, D) == 4 ? 2 : 1) void window_dkdv_pairs_kernel(WindowParams p) {
  using X = Tile<T, D>;
  constexpr int RT = 32, TB = X::bytes(RT), kPairs = key_pairs(T, D), KC = 32 * kPairs;
  __shared__ __align__(16) char lds[kSteps][2][TB];       // [which tile][queries, dout]
  __shared__ __align__(16) u32x4_t ops[2][kPairs][2 * X::C][64];  // p and dS of a step
  __shared__ float factors[2][kPairs][T == DSQG_F16 ? 64 : 1];    // ... dS's columns' factors
  __shared__ __align__(16) float rows[kSteps][3][RT];     // ... [reference exponent, 1 / sum, D]
  __shared__ int odd[kSteps][3];                          // ... queries, dout hold infinities or NaN; exponents are large
  static_assert(kSteps * 2 * TB >= kPairs * out_block<T, D>(), "the waves' output rows fit the tiles");

  const KeyBlock block(p);
  const int bk = block.bk, at = block.at, part = block.part;
  const int b = bk / p.Hkv, hk = bk - b * p.Hkv;
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = wave % kPairs;
  const bool maker = wave < kPairs;
  const int c = l & 31, h = l >> 5;
  const int length = window_length(p, b);
  const int k0 = at * KC, j0 = k0 + 32 * pair, j = j0 + c;

  int first, tiles;
  block.queries(p, RT, KC, length, first, tiles);
  const int steps = tiles * p.G;
  if (threadIdx.x < 3 * kSteps) odd[threadIdx.x / 3][threadIdx.x % 3] = 0;

  Stage<T, D, RT, 2 * 64 * kPairs> sq, sd;
  float2 st;
  float de;
  int lh = 0, li = 0;  // the next tile to load: its head and number
  auto load = [&] {
    const int head = hk * p.G + lh, i0 = (first + li) * RT;
    sq.load(p.q.at + b * p.q.b + head * p.q.h, p.q.n, i0, length);
    sd.load(p.dout.at + b * p.dout.b + head * p.dout.h, p.dout.n, i0, length);
    st = make_float2(INFINITY, 0.f);
    de = 0.f;
    if (threadIdx.x < RT && i0 + (int)threadIdx.x < length) {
      const long long s = ((long long)b * p.Hkv * p.G + head) * p.N + i0 + threadIdx.x;
      st = p.stats[s];
      de = p.delta[s];
    }
    if (++li == tiles) {
      li = 0;
      ++lh;
    }
  };
  auto store = [&](int t, int at, int i0) {  // step t's tile, whose first query is i0, to place `at`
    if (i0 < k0 + KC - 1 || (i0 + RT - 1 - k0 >= p.window && k0 + KC > p.sinks)) {  // some keys are not seen
      if (sq.clean()) odd[at][0] = t + 1;
      if (sd.clean()) odd[at][1] = t + 1;
    }
    sq.store(lds[at][0]);
    sd.store(lds[at][1]);
    if (threadIdx.x < RT) {
      rows[at][0][threadIdx.x] = st.x;
      rows[at][1][threadIdx.x] = st.y * weight_factor<T>();
      rows[at][2][threadIdx.x] = de;
      if (fabsf(st.x) >= kLarge && st.x != INFINITY) odd[at][2] = t + 1;
    }
  };
  auto next = [&](int x) { return x == kSteps - 1 ? 0 : x + 1; };
  // Nothing of the tile from query i0 on sees the wave's keys.
  auto none = [&](int i0) { return i0 + 31 < j0 || (i0 - (j0 + 31) >= p.window && j0 >= p.sinks); };
  auto seen_of = [&](int i0) {  // (Rows are queries here: a sink is seen by all from itself on.)
    return Seen{j - i0, j < p.sinks ? 64 : min(64, j - i0 + p.window - 1), 0};
  };

  __syncthreads();
  if (steps > 0) {
    load();
    store(0, 0, first * RT);
    if (steps > 1) load();
  }
  __syncthreads();

  if (maker) {
    u32x4_t k[X::KS], v[X::KS];
    {
      const char* const rk = p.k.at + b * p.k.b + hk * p.k.h + (long long)j * p.k.n;
      const char* const rv = p.v.at + b * p.v.b + hk * p.v.h + (long long)j * p.v.n;
#pragma unroll
      for (int s = 0; s < X::KS; ++s) {
        const int e = (2 * X::E * s + X::E * h) * X::O::size;
        k[s] = frag_or_zero(rk + e, j < length);
        v[s] = frag_or_zero(rv + e, j < length);
      }
    }
    int place = 0, tile = 0;
    float factor = T == DSQG_F16 ? kNoFactor : 1.f;
#pragma unroll 1
    for (int t = 0; t <= steps; ++t) {
      const int i0 = (first + tile) * RT;
      if (t < steps && !none(i0)) {
        const char* const qt = lds[place][0];
        const char* const dt = lds[place][1];
        const f32x16_t s = scores<T, D>(qt, l, k), dp = scores<T, D>(dt, l, v);
        const bool large = odd[place][2] == t + 1;
        float w[16], x[16], m[16];
#pragma unroll
        for (int r4 = 0; r4 < 16; r4 += 4) {
          const f32x4_t y = *reinterpret_cast<const f32x4_t*>(&rows[place][0][reg_row<T>(r4, h)]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[r4 + e] = s[r4 + e];
            m[r4 + e] = y[e];
          }
        }
        exponents(w, p.scale2, large, [&](int r) { return m[r]; });
#pragma unroll
        for (int r4 = 0; r4 < 16; r4 += 4) {
          const int row = reg_row<T>(r4, h);
          const f32x4_t y = *reinterpret_cast<const f32x4_t*>(&rows[place][1][row]);
          const f32x4_t d = *reinterpret_cast<const f32x4_t*>(&rows[place][2][row]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[r4 + e] = __builtin_amdgcn_exp2f(w[r4 + e]) * y[e];
            x[r4 + e] = w[r4 + e] * (dp[r4 + e] - d[e]);
          }
        }
        const bool all = i0 >= j0 + 31 && (i0 + 31 - j0 < p.window || j0 + 32 <= p.sinks);
        if (!all) hide<T>(0.f, seen_of(i0), false, h, w, x);
        Weights<T> f;
        pack<T>(w, f);
#pragma unroll
        for (int e = 0; e < X::C; ++e) ops[t & 1][pair][e][l] = f[e];
        if constexpr (T == DSQG_F16) {
          factor = next_factor(x, factor);
          factors[t & 1][pair][l] = factor;
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] *= factor;
        }
        pack<T>(x, f);
#pragma unroll
        for (int e = 0; e < X::C; ++e) ops[t & 1][pair][X::C + e][l] = f[e];
      }
      place = next(place);
      if (++tile == tiles) tile = 0;
      if (t + 1 < steps) {
        store(t + 1, place, (first + tile) * RT);
        if (t + 2 < steps) load();
      }
      __syncthreads();
    }
    return;
  }

  Acc<T, D> dk, dv;
#pragma unroll
  for (int d = 0; d < X::DB; ++d) dk[d] = dv[d] = zero_tile();
  float factor = T == DSQG_F16 ? kNoFactor : 1.f;
  int place = 0, last = 0, tile = 0, was = 0, head = hk * p.G;  // of step t, and of the step before
#pragma unroll 1
  for (int t = 0; t <= steps; ++t) {
    const int i0 = (first + was) * RT;
    if (t > 0 && !none(i0)) {
      const char* const qt = lds[last][0];
      const char* const dt = lds[last][1];
      Weights<T> f;
#pragma unroll
      for (int e = 0; e < X::C; ++e) f[e] = ops[(t - 1) & 1][pair][e][l];
      contract<T, D>(dv, dt, l, f);
#pragma unroll
      for (int e = 0; e < X::C; ++e) f[e] = ops[(t - 1) & 1][pair][X::C + e][l];
      if constexpr (T == DSQG_F16) refactor(dk, factor, factors[(t - 1) & 1][pair][l]);
      contract<T, D>(dk, qt, l, f);
      if (odd[last][0] == t)
        add_odd<T, D>(dk, p.q.at + b * p.q.b + head * p.q.h + i0 * p.q.n, p.q.n, length - i0, l, seen_of(i0));
      if (odd[last][1] == t)
        add_odd<T, D>(dv, p.dout.at + b * p.dout.b + head * p.dout.h + i0 * p.dout.n, p.dout.n, length - i0, l, seen_of(i0));
    }
    if (t > 0 && was == tiles - 1) ++head;
    was = tile;
    last = place;
    place = next(place);
    if (++tile == tiles) tile = 0;
    if (t + 1 < steps) {
      store(t + 1, place, (first + tile) * RT);
      if (t + 2 < steps) load();
    }
    __syncthreads();
  }

  const float fk = unfactor(factor, 1.f / weight_factor<T>()), fv = 1.f / weight_factor<T>();
  if (at < p.split) {
    float* const to = p.part + ((((long long)bk * p.split + at) * (1 + p.far) + part) * 2 * KC + 32 * pair + c) * D;
#pragma unroll
    for (int d = 0; d < X::DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = 32 * d + 8 * g + 4 * h;
        if (D % 32 != 0 && e >= D) continue;
        *reinterpret_cast<f32x4_t*>(to + e) = f32x4_t{dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]} * fk;
        *reinterpret_cast<f32x4_t*>(to + KC * D + e) = f32x4_t{dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]} * fv;
      }
    return;
  }
  char* const mine = lds[0][0] + pair * out_block<T, D>();
  store_columns<T, D>(dk, fk * p.scale, j < length, mine, p.dk.at + b * p.dk.b + hk * p.dk.h + j0 * p.dk.n, p.dk.n, p.N - j0, l);
  store_columns<T, D>(dv, fv, j < length, mine, p.dv.at + b * p.dv.b + hk * p.dv.h + j0 * p.dv.n, p.dv.n, p.N - j0, l);
}

// Sums of the sinks' key blocks over their parts.  Grid: [B * Hkv * split * kcols / 8, 2], a thread four elements.
template <int T, int D>
__global__ __launch_bounds__(kBlock) void window_sinks_kernel(WindowParams p) {
  constexpr int L = D / 4;  // lanes of a row
  const int which = blockIdx.y;
  for (int e = threadIdx.x; e < 8 * L; e += kBlock) {
    const long long row = (long long)blockIdx.x * 8 + e / L;
    const int col = (int)(row % p.kcols), d = e % L * 4;
    const long long block = row / p.kcols;
    const int at = (int)(block % p.split), bk = (int)(block / p.split), b = bk / p.Hkv, hk = bk - b * p.Hkv, j = at * p.kcols + col;
    if (j >= p.N) continue;
    f32x4_t x = zero4();
    const float* from = p.part + ((block * (1 + p.far) * 2 + which) * p.kcols + col) * D + d;
    const int parts = j < p.sinks ? p.far : 0;  // (others' keys are not seen from afar)
    // (Sixteen parts' loads at once: 4.6 us at D = 32 with 18 far parts, 5.6 at D = 128 with 53;
    // one after the other 7.9 and 15.7.)
    constexpr int kAtOnce = 16;
    for (int i = 0; i <= parts; i += kAtOnce) {
      f32x4_t y[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        y[u] = *reinterpret_cast<const f32x4_t*>(from + (long long)min(i + u, parts) * 2 * p.kcols * D);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (i + u <= parts) x += y[u];
    }
    const bool live = j < window_length(p, b);
    const float f = which == 0 ? p.scale : 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = live ? x[i] * f : 0.f;
    const WindowRows& o = which == 0 ? p.dk : p.dv;
    char* const to = o.at + b * o.b + hk * o.h + j * o.n + d * Op<T>::size;
    if constexpr (T == DSQG_F32) {
      *reinterpret_cast<f32x4_t*>(to) = x;
    } else if constexpr (T == DSQG_BF16) {
      *reinterpret_cast<uint2*>(to) = make_uint2(cvt_pk_bf16(x[0], x[1]), cvt_pk_bf16(x[2], x[3]));
    } else {
      *reinterpret_cast<uint2*>(to) = make_uint2(__builtin_bit_cast(uint32_t, half2_t{(_Float16)x[0], (_Float16)x[1]}),
                                                 __builtin_bit_cast(uint32_t, half2_t{(_Float16)x[2], (_Float16)x[3]}));
    }
  }
}

template <int T, int D>
hipError_t launch(const WindowParams& p, hipStream_t st) {
  const unsigned heads = (unsigned)(p.B * p.Hkv), blocks = heads * (unsigned)(p.G * p.blocks);
  bool wide = false;
  if constexpr (may_be_wide(T, D)) {
    wide = p.waves == 8;
    if (wide) hipLaunchKernelGGL((window_dq_kernel<T, D, 8>), dim3(blocks), dim3(512), 0, st, p);
  }
  if (!wide) hipLaunchKernelGGL((window_dq_kernel<T, D, 4>), dim3(blocks), dim3(256), 0, st, p);
  const dim3 grid(heads * (unsigned)(p.kblocks + p.split * p.far));
  if constexpr (D > kSingle) hipLaunchKernelGGL((window_dkdv_pairs_kernel<T, D>), grid, dim3(dkdv_threads<T, D>()), 0, st, p);
  else hipLaunchKernelGGL((window_dkdv_kernel<T, D>), grid, dim3(kBlock), 0, st, p);
  if (p.split)
    hipLaunchKernelGGL((window_sinks_kernel<T, D>), dim3(heads * (unsigned)(p.split * p.kcols / 8), 2), dim3(kBlock), 0, st, p);
  return hipGetLastError();
}

template <int T>
hipError_t launch_dim(const WindowParams& p, hipStream_t st) {
  switch (p.D) {
    case 32: return launch<T, 32>(p, st);
    case 64: return launch<T, 64>(p, st);
    case 80: return launch<T, 80>(p, st);
    case 96: return launch<T, 96>(p, st);
    default: return launch<T, 128>(p, st);
  }
}

}  // namespace

hipError_t launch_window_bwd(const WindowParams& p, int dtype, hipStream_t st) {
  if (dtype == DSQG_F32) return launch_dim<DSQG_F32>(p, st);
  if (dtype == DSQG_BF16) return launch_dim<DSQG_BF16>(p, st);
  return launch_dim<DSQG_F16>(p, st);
}

namespace {

// The checks that all entry points share, and the split.
int check_window(const dsqg_window_shape& s, WindowParams* p, bool backward) {
  if (s.dtype != DSQG_F32 && s.dtype != DSQG_BF16 && s.dtype != DSQG_F16) return DSQG_EINVAL;
  if (s.B < 0 || s.H < 0 || s.Hkv < 0 || s.N < 0 || s.D <= 0 || s.window < 1 || s.sinks < 0) return DSQG_EINVAL;
  if (s.Hkv > 0 ? s.H == 0 || s.H % s.Hkv != 0 : s.H != 0) return DSQG_EINVAL;
  if (!head_dim_supported(s.D)) return DSQG_EUNSUPPORTED;
  *p = WindowParams{};
  p->B = s.B; p->Hkv = s.Hkv; p->N = s.N; p->D = s.D;
  if (s.B == 0 || s.H == 0 || s.N == 0) return DSQG_OK;
  // Positions plus a window are 32 bits, grids less than 2^32 lanes.
  constexpr long long lanes = 1ll << 32;
  if (s.N > (1 << 30) || (long long)s.B * s.H >= lanes / 256) return DSQG_EUNSUPPORTED;
  p->G = s.H / s.Hkv;
  p->window = std::min(s.window, 1 << 30);
  p->sinks = std::min(s.sinks, 1 << 30);
  p->scale = s.softmax_scale;
  // (No scale gives equal weights to all scores up to 2^100, and a score of -infinity none.)
  p->scale2 = s.softmax_scale == 0.f ? 0x1p-126f : s.softmax_scale * 1.4426950408889634f;
  p->lengths = reinterpret_cast<const long long*>(s.lengths);
  // Eight waves of 32 queries share a tile where that leaves two workgroups for each CU, else four (may_be_wide).
  p->waves = may_be_wide(s.dtype, s.D) && (long long)s.B * s.H * ((s.N + 255ll) / 256) >= 512 ? 8 : 4;
  p->blocks = (s.N + 32 * p->waves - 1) / (32 * p->waves);
  if ((long long)s.B * s.H * p->blocks * (64 * p->waves) >= lanes) return DSQG_EUNSUPPORTED;
  // The sinks' far queries: shares of a quarter of the queries that other blocks see, which fill the places that those leave
  // free at the end; 64 of them at most.
  const int kc = p->kcols = 32 * key_pairs(s.dtype, s.D);
  p->kblocks = (s.N + kc - 1) / kc;
  const long long beyond = (long long)s.N - kc - p->window;
  if (p->sinks > 0 && beyond > 0) {
    p->split = (std::min(p->sinks, s.N) + kc - 1) / kc;
    const long long share = std::max(64, (p->window + kc) / 4);
    p->far = (int)std::min((beyond + share - 1) / share, std::max(1ll, 64ll / p->split));
  }
  if (backward) {
    const long long heads = (long long)s.B * s.Hkv, threads = s.D > kSingle ? 4 * kc : kBlock;
    if (heads * (p->kblocks + (long long)p->split * p->far) * threads >= lanes || heads * p->split * (kc / 8) * kBlock >= lanes)
      return DSQG_EUNSUPPORTED;
  }
  return DSQG_OK;
}

size_t delta_bytes(const dsqg_window_shape& s) { return ((size_t)s.B * s.H * s.N * sizeof(float) + 255) / 256 * 256; }
size_t part_bytes(const WindowParams& p) {
  return (size_t)p.B * p.Hkv * p.split * (1 + p.far) * 2 * p.kcols * p.D * sizeof(float);
}

// Rows: a base and strides {b, h, n} that keep every row 16-byte aligned, and rows that do not overlap, within 2^24 bytes.
bool rows_of(const void* ptr, const int64_t st[3], int dtype, int D, int N, WindowRows* r) {
  const long long es = dtype == DSQG_F32 ? 4 : 2;
  if (!ptr || (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (st[i] < 0 || st[i] > (1ll << 50) || st[i] * es % 16 != 0) return false;
  if (N > 1 && (st[2] < D || st[2] * es >= (1 << 24))) return false;
  r->at = static_cast<char*>(const_cast<void*>(ptr));
  r->b = st[0] * es; r->h = st[1] * es; r->n = N > 1 ? st[2] * es : D * es;
  return true;
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" int dsqg_window_fwd(const dsqg_window_fwd_args* a, dsqg_stream_t stream) {
  if (!a) return DSQG_EINVAL;
  WindowParams p;
  const dsqg_window_shape& s = a->shape;
  if (const int st = check_window(s, &p, false)) return st;
  if (s.B == 0 || s.H == 0 || s.N == 0) return DSQG_OK;
  auto rows = [&](const void* ptr, const int64_t st[3], WindowRows* r) { return rows_of(ptr, st, s.dtype, s.D, s.N, r); };
  if (!rows(a->q, a->q_stride, &p.q) || !rows(a->k, a->k_stride, &p.k) || !rows(a->v, a->v_stride, &p.v) ||
      !rows(a->out, a->out_stride, &p.out) || (reinterpret_cast<uintptr_t>(a->stats) & 7u) != 0)
    return DSQG_EINVAL;
  p.stats = reinterpret_cast<float2*>(a->stats);
  if (a->low && (s.dtype == DSQG_F32 || !rows(a->low, a->low_stride, &p.low))) return DSQG_EINVAL;
  return launch_window_fwd(p, s.dtype, reinterpret_cast<hipStream_t>(stream)) == hipSuccess ? DSQG_OK : DSQG_EHIP;
}

extern "C" int dsqg_window_bwd_workspace_size(const dsqg_window_shape* s, size_t* bytes) {
  WindowParams p;
  if (!s || !bytes) return DSQG_EINVAL;
  if (const int st = check_window(*s, &p, true)) return st;
  *bytes = s->B == 0 || s->H == 0 || s->N == 0 ? 0 : delta_bytes(*s) + part_bytes(p);
  return DSQG_OK;
}

extern "C" int dsqg_window_bwd(const dsqg_window_bwd_args* a, dsqg_stream_t stream) {
  if (!a) return DSQG_EINVAL;
  WindowParams p;
  const dsqg_window_shape& s = a->shape;
  if (const int st = check_window(s, &p, true)) return st;
  if (s.B == 0 || s.H == 0 || s.N == 0) return DSQG_OK;
  auto rows = [&](const void* ptr, const int64_t st[3], WindowRows* r) { return rows_of(ptr, st, s.dtype, s.D, s.N, r); };
  if (!rows(a->q, a->q_stride, &p.q) || !rows(a->k, a->k_stride, &p.k) || !rows(a->v, a->v_stride, &p.v) ||
      !rows(a->out, a->out_stride, &p.out) || !rows(a->dout, a->dout_stride, &p.dout) || !rows(a->dq, a->dq_stride, &p.dq) ||
      !rows(a->dk, a->dk_stride, &p.dk) || !rows(a->dv, a->dv_stride, &p.dv) || !a->stats ||
      (reinterpret_cast<uintptr_t>(a->stats) & 7u) != 0)
    return DSQG_EINVAL;
  if (a->low && (s.dtype == DSQG_F32 || !rows(a->low, a->low_stride, &p.low))) return DSQG_EINVAL;
  if (!a->workspace || a->workspace_bytes < delta_bytes(s) + part_bytes(p)) return DSQG_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return DSQG_EINVAL;
  p.stats = reinterpret_cast<float2*>(const_cast<float*>(a->stats));
  p.delta = static_cast<float*>(a->workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + delta_bytes(s));
  return launch_window_bwd(p, s.dtype, reinterpret_cast<hipStream_t>(stream)) == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
