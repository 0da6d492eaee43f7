// Attention within a window and its sinks, backward (gfx950).
//
//   p_ij = 2^(scale2 q_i.k_j - m_i) / sum_i,   D_i = dout_i . out_i,   dS_ij = p_ij (dout_i . v_j - D_i)
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
// p and dS enter the products rounded to the 16-bit type (2^-8 of each in bfloat16, 2^-11 in float16); float32 operands are not
// rounded.  Everything else is fp32.
#include <algorithm>

#include "dsqg_window.hpp"

namespace dsqg {
namespace {

template <int T, int D> constexpr int rows_of_tile() { return T == DSQG_F32 || D > 64 ? 32 : 64; }

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

template <int T, int D>
__global__ __launch_bounds__(kBlock, 2) void window_dq_kernel(WindowParams p) {
  using X = Tile<T, D>;
  constexpr int RT = rows_of_tile<T, D>(), KB = RT / 32, TB = X::bytes(RT);
  __shared__ __align__(16) char lds[2][2][TB];
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
  float delta = 0.f;
  {
    const char* const rq = p.q.at + b * p.q.b + head * p.q.h + (long long)i * p.q.n;
    const char* const rd = p.dout.at + b * p.dout.b + head * p.dout.h + (long long)i * p.dout.n;
    const char* const ro = p.out.at + b * p.out.b + head * p.out.h + (long long)i * p.out.n;
#pragma unroll
    for (int s = 0; s < X::KS; ++s) {
      const int e = (2 * X::E * s + X::E * h) * X::O::size;
      q[s] = frag_or_zero(rq + e, i < length);
      dout[s] = frag_or_zero(rd + e, i < length);
      delta = dot_frag<T>(dout[s], frag_or_zero(ro + e, i < length), delta);
    }
    delta = xor32_pair_sum(delta);
  }
  float2 st = make_float2(INFINITY, 0.f);
  if (i < length) st = p.stats[stat];
  const bool large = __any(i < length && fabsf(st.x) >= kLarge);
  if (h == 0 && i < p.N) p.delta[stat] = delta;
  if (threadIdx.x < 2) odd[threadIdx.x] = 0;

  Stage<T, D, RT> sk, sv;
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
      const char* const kt = lds[t & 1][0] + 32 * kb * X::RV * X::O::size;
      const char* const vt = lds[t & 1][1] + 32 * kb * X::RV * X::O::size;
      f32x16_t s = zero_tile(), dp = zero_tile();
#pragma unroll
      for (int e = 0; e < X::KS; ++e) s = mma<T>(row_frag<T, D>(kt, l, e), q[e], s);
#pragma unroll
      for (int e = 0; e < X::KS; ++e) dp = mma<T>(row_frag<T, D>(vt, l, e), dout[e], dp);
      auto sees = [&](int row) {
        const int back = i - (k0 + row);
        return back >= 0 && (back < p.window || k0 + row < p.sinks);
      };
      float w[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = exponent(s[r], p.scale2, st.x, large);
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = __builtin_amdgcn_exp2f(w[r]) * st.y * (dp[r] - delta);
      if (!all) {
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] = sees(reg_row<T>(r, h)) ? w[r] : 0.f;
      }
      Weights<T> f;
      pack<T>(w, f);
      contract<T, D>(acc, kt, l, f);
      if (odd[t & 1] == t + 1) add_odd<T, D>(acc, kh + k0 * p.k.n, p.k.n, length - k0, l, sees);
    }
    if (t + 1 < span.n) {
      store(t + 1);
      if (t + 2 < span.n) load(t + 2);
    }
    __syncthreads();
  }
  store_columns<T, D>(acc, p.scale, i < length, lds[0][0] + wave * 32 * X::RV * X::O::size,
                      p.dq.at + b * p.dq.b + head * p.dq.h + i0 * p.dq.n, p.dq.n, p.N - i0, l);
}

template <int T, int D>
__global__ __launch_bounds__(kBlock) void window_dkdv_kernel(WindowParams p) {
  using X = Tile<T, D>;
  constexpr int RT = rows_of_tile<T, D>(), RB = RT / 32, TB = X::bytes(RT);
  __shared__ __align__(16) char lds[2][2][TB];         // [which tile][queries, dout]
  __shared__ __align__(16) float rows[2][3][RT];       // ... [reference exponent, 1 / sum, D]
  __shared__ int odd[2][3];                            // ... queries, dout hold infinities or NaN; exponents are large

  const int roles = p.blocks + p.split * p.far;  // of a key/value head; those of the sinks' far queries first
  const int block = xcd_logical_block(blockIdx.x, gridDim.x);
  const int bk = block / roles, role = block - bk * roles;
  const int b = bk / p.Hkv, hk = bk - b * p.Hkv;
  const int at = role < p.split * p.far ? role / p.far : role - p.split * p.far;
  const int part = role < p.split * p.far ? 1 + role % p.far : 0;
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = l & 31, h = l >> 5;
  const int length = window_length(p, b);
  const int k0 = at * kCols, j0 = k0 + 32 * wave, j = j0 + c;

  // Tiles of queries: of each head the same.
  int first = k0 / RT, tiles = 0;
  if (k0 < length) {
    const int last = (length - 1) / RT;
    const int near = min((long long)last, ((long long)k0 + kCols - 2 + p.window) / RT);  // of the window
    if (at >= p.split) tiles = (k0 < p.sinks ? last : near) + 1 - first;
    else if (part == 0) tiles = near + 1 - first;
    else {
      const int n = last - near, lo = (int)((long long)n * (part - 1) / p.far), hi = (int)((long long)n * part / p.far);
      first = near + 1 + lo;
      tiles = hi - lo;
    }
  }
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
    return i0 < k0 + kCols - 1 || (i0 + RT - 1 - k0 >= p.window && k0 + kCols > p.sinks);
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
      rows[t & 1][1][threadIdx.x] = st.y;
      rows[t & 1][2][threadIdx.x] = de;
      if (fabsf(st.x) >= kLarge && st.x != INFINITY) odd[t & 1][2] = t + 1;
    }
  };

  Acc<T, D> dk, dv;
#pragma unroll
  for (int d = 0; d < X::DB; ++d) dk[d] = dv[d] = zero_tile();

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
      const char* const qt = lds[t & 1][0] + 32 * rb * X::RV * X::O::size;
      const char* const dt = lds[t & 1][1] + 32 * rb * X::RV * X::O::size;
      auto sees = [&](int row) {
        const int back = i0 + row - j;
        return back >= 0 && (back < p.window || j < p.sinks);
      };
      f32x16_t s = zero_tile(), dp = zero_tile();
#pragma unroll
      for (int e = 0; e < X::KS; ++e) s = mma<T>(row_frag<T, D>(qt, l, e), k[e], s);
#pragma unroll
      for (int e = 0; e < X::KS; ++e) dp = mma<T>(row_frag<T, D>(dt, l, e), v[e], dp);
      const bool large = odd[t & 1][2] == t + 1;
      float w[16], x[16];
#pragma unroll
      for (int r4 = 0; r4 < 16; r4 += 4) {
        const int row = 32 * rb + reg_row<T>(r4, h);
        const f32x4_t m = *reinterpret_cast<const f32x4_t*>(&rows[t & 1][0][row]);
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(&rows[t & 1][1][row]);
        const f32x4_t d = *reinterpret_cast<const f32x4_t*>(&rows[t & 1][2][row]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[r4 + e] = __builtin_amdgcn_exp2f(exponent(s[r4 + e], p.scale2, m[e], large)) * y[e];
          x[r4 + e] = w[r4 + e] * (dp[r4 + e] - d[e]);
        }
      }
      if (!all) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool seen = sees(reg_row<T>(r, h));
          w[r] = seen ? w[r] : 0.f;
          x[r] = seen ? x[r] : 0.f;
        }
      }
      Weights<T> f;
      pack<T>(w, f);
      contract<T, D>(dv, dt, l, f);
      pack<T>(x, f);
      contract<T, D>(dk, qt, l, f);
      const int head = hk * p.G + t / tiles;
      if (odd[t & 1][0] == t + 1)
        add_odd<T, D>(dk, p.q.at + b * p.q.b + head * p.q.h + i0 * p.q.n, p.q.n, length - i0, l, sees);
      if (odd[t & 1][1] == t + 1)
        add_odd<T, D>(dv, p.dout.at + b * p.dout.b + head * p.dout.h + i0 * p.dout.n, p.dout.n, length - i0, l, sees);
    }
    if (t + 1 < steps) {
      store(t + 1);
      if (t + 2 < steps) load(t + 2);
    }
    __syncthreads();
  }

  if (at < p.split) {
    float* const to = p.part + ((((long long)bk * p.split + at) * (1 + p.far) + part) * 2 * kCols + 32 * wave + c) * D;
#pragma unroll
    for (int d = 0; d < X::DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = 32 * d + 8 * g + 4 * h;
        if (D % 32 != 0 && e >= D) continue;
        *reinterpret_cast<f32x4_t*>(to + e) = f32x4_t{dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]};
        *reinterpret_cast<f32x4_t*>(to + kCols * D + e) = f32x4_t{dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]};
      }
    return;
  }
  char* const mine = lds[0][0] + wave * 32 * X::RV * X::O::size;
  store_columns<T, D>(dk, p.scale, j < length, mine, p.dk.at + b * p.dk.b + hk * p.dk.h + j0 * p.dk.n, p.dk.n, p.N - j0, l);
  store_columns<T, D>(dv, 1.f, j < length, mine, p.dv.at + b * p.dv.b + hk * p.dv.h + j0 * p.dv.n, p.dv.n, p.N - j0, l);
}

// Sums of the sinks' key blocks over their parts.  Grid: [B * Hkv * split * kCols / 8, 2], a thread four elements.
template <int T, int D>
__global__ __launch_bounds__(kBlock) void window_sinks_kernel(WindowParams p) {
  constexpr int L = D / 4;  // lanes of a row
  const int which = blockIdx.y;
  for (int e = threadIdx.x; e < 8 * L; e += kBlock) {
    const long long row = (long long)blockIdx.x * 8 + e / L;
    const int col = (int)(row % kCols), d = e % L * 4;
    const long long block = row / kCols;
    const int at = (int)(block % p.split), bk = (int)(block / p.split), b = bk / p.Hkv, hk = bk - b * p.Hkv, j = at * kCols + col;
    if (j >= p.N) continue;
    f32x4_t x = zero4();
    const float* from = p.part + ((block * (1 + p.far) * 2 + which) * kCols + col) * D + d;
    for (int i = 0; i <= p.far; ++i) x += *reinterpret_cast<const f32x4_t*>(from + (long long)i * 2 * kCols * D);
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
  const unsigned heads = (unsigned)(p.B * p.Hkv);
  hipLaunchKernelGGL((window_dq_kernel<T, D>), dim3(heads * (unsigned)(p.G * p.blocks)), dim3(kBlock), 0, st, p);
  hipLaunchKernelGGL((window_dkdv_kernel<T, D>), dim3(heads * (unsigned)(p.blocks + p.split * p.far)), dim3(kBlock), 0, st, p);
  if (p.split)
    hipLaunchKernelGGL((window_sinks_kernel<T, D>), dim3(heads * (unsigned)(p.split * kCols / 8), 2), dim3(kBlock), 0, st, p);
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

// The checks that all entry points share.
int check_window(const dsqg_window_shape& s, WindowParams* p) {
  if (s.dtype != DSQG_F32 && s.dtype != DSQG_BF16 && s.dtype != DSQG_F16) return DSQG_EINVAL;
  if (s.B < 0 || s.H < 0 || s.Hkv < 0 || s.N < 0 || s.D <= 0 || s.window < 1 || s.sinks < 0) return DSQG_EINVAL;
  if (s.Hkv > 0 ? s.H == 0 || s.H % s.Hkv != 0 : s.H != 0) return DSQG_EINVAL;
  if (!head_dim_supported(s.D)) return DSQG_EUNSUPPORTED;
  *p = WindowParams{};
  p->B = s.B; p->Hkv = s.Hkv; p->N = s.N; p->D = s.D;
  if ((long long)s.B * s.H * s.N == 0) return DSQG_OK;
  p->G = s.H / s.Hkv;
  p->window = std::min(s.window, 1 << 30);
  p->sinks = std::min(s.sinks, 1 << 30);
  p->scale = s.softmax_scale;
  p->scale2 = s.softmax_scale * 1.4426950408889634f;
  p->lengths = reinterpret_cast<const long long*>(s.lengths);
  p->blocks = (s.N + kCols - 1) / kCols;
  // The grids, and positions plus a window in 32 bits.
  if (s.N > (1 << 30) || (long long)s.B * s.H * (p->blocks + 64) >= (1ll << 31)) return DSQG_EUNSUPPORTED;
  // The sinks' far queries: shares of about as many queries as the other blocks see, 64 of them at most.
  const long long beyond = (long long)s.N - kCols - p->window;
  if (p->sinks > 0 && beyond > 0) {
    p->split = (std::min(p->sinks, s.N) + kCols - 1) / kCols;
    p->far = (int)std::min((beyond + p->window + kCols - 1) / (p->window + kCols), std::max(1ll, 64ll / p->split));
  }
  return DSQG_OK;
}

size_t delta_bytes(const dsqg_window_shape& s) { return ((size_t)s.B * s.H * s.N * sizeof(float) + 255) / 256 * 256; }
size_t part_bytes(const WindowParams& p) {
  return (size_t)p.B * p.Hkv * p.split * (1 + p.far) * 2 * kCols * p.D * sizeof(float);
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
  if (const int st = check_window(s, &p)) return st;
  if ((long long)s.B * s.H * s.N == 0) return DSQG_OK;
  auto rows = [&](const void* ptr, const int64_t st[3], WindowRows* r) { return rows_of(ptr, st, s.dtype, s.D, s.N, r); };
  if (!rows(a->q, a->q_stride, &p.q) || !rows(a->k, a->k_stride, &p.k) || !rows(a->v, a->v_stride, &p.v) ||
      !rows(a->out, a->out_stride, &p.out) || (reinterpret_cast<uintptr_t>(a->stats) & 7u) != 0)
    return DSQG_EINVAL;
  p.stats = reinterpret_cast<float2*>(a->stats);
  return launch_window_fwd(p, s.dtype, reinterpret_cast<hipStream_t>(stream)) == hipSuccess ? DSQG_OK : DSQG_EHIP;
}

extern "C" int dsqg_window_bwd_workspace_size(const dsqg_window_shape* s, size_t* bytes) {
  WindowParams p;
  if (!s || !bytes) return DSQG_EINVAL;
  if (const int st = check_window(*s, &p)) return st;
  *bytes = (long long)s->B * s->H * s->N == 0 ? 0 : delta_bytes(*s) + part_bytes(p);
  return DSQG_OK;
}

extern "C" int dsqg_window_bwd(const dsqg_window_bwd_args* a, dsqg_stream_t stream) {
  if (!a) return DSQG_EINVAL;
  WindowParams p;
  const dsqg_window_shape& s = a->shape;
  if (const int st = check_window(s, &p)) return st;
  if ((long long)s.B * s.H * s.N == 0) return DSQG_OK;
  auto rows = [&](const void* ptr, const int64_t st[3], WindowRows* r) { return rows_of(ptr, st, s.dtype, s.D, s.N, r); };
  if (!rows(a->q, a->q_stride, &p.q) || !rows(a->k, a->k_stride, &p.k) || !rows(a->v, a->v_stride, &p.v) ||
      !rows(a->out, a->out_stride, &p.out) || !rows(a->dout, a->dout_stride, &p.dout) || !rows(a->dq, a->dq_stride, &p.dq) ||
      !rows(a->dk, a->dk_stride, &p.dk) || !rows(a->dv, a->dv_stride, &p.dv) || !a->stats ||
      (reinterpret_cast<uintptr_t>(a->stats) & 7u) != 0)
    return DSQG_EINVAL;
  if (!a->workspace || a->workspace_bytes < delta_bytes(s) + part_bytes(p)) return DSQG_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return DSQG_EINVAL;
  p.stats = reinterpret_cast<float2*>(const_cast<float*>(a->stats));
  p.delta = static_cast<float*>(a->workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + delta_bytes(s));
  return launch_window_bwd(p, s.dtype, reinterpret_cast<hipStream_t>(stream)) == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
