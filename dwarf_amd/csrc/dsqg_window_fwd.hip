// Attention within a window and its sinks, forward (gfx950).
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j     over the positions j that i sees (dsqg_window.hpp)
//
// A workgroup takes 128 or 256 queries of a head, a wave 32 of them, and goes once over the tiles of keys and values that any of
// them sees, with a running maximum and sum: S^T = K Q^T, weights, O^T += V^T P^T, the weights staying in registers from
// one product to the other.  Keys and values are loaded a tile ahead and lie in LDS twice, so that a tile costs one
// barrier.  Only tiles at the window's two ends (and the sinks') compare positions.
//
// Weights are rounded once to the 16-bit type before they multiply the values (2^-8 of each in bfloat16, 2^-11 in float16); float32
// operands are not rounded.  Scores, the maximum, the sum and the output's sums are fp32.  For the backward a query's
// reference exponent m and 1 / sum are kept apart, for m may be too large to hold the sum's logarithm.
//
// Measured (bfloat16): B1 H16 Hkv4 N16384 D128 window 1024, 240 us, 570 TFLOP/s of the two products; B8 H8 Hkv8 N2048 D32 window
// 256 with 4 sinks, 24 us, 190 TFLOP/s.  Vector instructions and latency bound it: at D = 128 46 % of the cycles issue
// vector work and 21 % matrix work, at D = 32 a score costs as many vector instructions for a quarter of the products.
#include "dsqg_window.hpp"

namespace dsqg {
namespace {

// One pass of workgroup `workgroup`, with values times 2^-30 where `small`; says whether one of its sums was no number, with
// nothing written.
template <int T, int D, int NW>
__device__ __forceinline__ bool window_fwd_pass(const WindowParams& p, int workgroup, int thread, bool small) {
  using X = Tile<T, D>;
  constexpr int RT = T == DSQG_F32 || (D > 64 && NW == 4) ? 32 : 64, KB = RT / 32, TB = X::bytes(RT), kCols = 32 * NW;
  constexpr int BYTES = 4 * TB > NW * out_block<T, D>() ? 4 * TB : NW * out_block<T, D>();
  __shared__ __align__(16) char bytes[BYTES];          // the tiles, in the end the waves' output rows
  auto lds = reinterpret_cast<char(*)[2][TB]>(bytes);  // [which tile][keys, values]
  __shared__ int odd[2];                        // which tile's values hold infinities or NaN, plus one
  __shared__ int over;                          // whether a sum is no number

  // Blocks that read the same keys, the heads of a key/value head, follow each other; the longest come first.
  const int block = xcd_logical_block(workgroup, gridDim.x);
  const int g = block % p.G, rest = block / p.G;
  const int at = p.blocks - 1 - rest % p.blocks, bk = rest / p.blocks;
  const int b = bk / p.Hkv, hk = bk - b * p.Hkv, head = hk * p.G + g;
  const int l = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
  const int c = l & 31, h = l >> 5;
  const int length = window_length(p, b);
  const int q0 = at * kCols, i0 = q0 + 32 * wave, i = i0 + c;
  const char* const kh = p.k.at + b * p.k.b + hk * p.k.h;
  const char* const vh = p.v.at + b * p.v.b + hk * p.v.h;
  const WindowSpan span = q0 < length ? keys_of<RT>(p, q0, min(q0 + kCols, length) - 1) : WindowSpan{0, 0, 0};

  u32x4_t q[X::KS];
  {
    const char* const row = p.q.at + b * p.q.b + head * p.q.h + (long long)i * p.q.n;
#pragma unroll
    for (int s = 0; s < X::KS; ++s) {
      q[s] = u32x4_t{0u, 0u, 0u, 0u};
      if (i < length) q[s] = *reinterpret_cast<const u32x4_t*>(row + (2 * X::E * s + X::E * h) * X::O::size);
    }
  }
  if (thread < 2) odd[thread] = 0;
  // (A second pass leaves it: slower waves may still be about to read it.)
  if (thread == 0 && !small) over = 0;

  Stage<T, D, RT, 64 * NW> sk, sv;
  auto load = [&](int t) {
    sk.load(kh, p.k.n, span.tile(t) * RT, length);
    sv.load(vh, p.v.n, span.tile(t) * RT, length);
  };
  // Whether some of the workgroup's queries do not see some of tile t.
  auto edge = [&](int t) {
    const int j0 = span.tile(t) * RT;
    return j0 + RT - 1 > q0 || (q0 + kCols - 1 - j0 >= p.window && j0 + RT > p.sinks);
  };
  auto store = [&](int t) {
    sk.store(lds[t & 1][0]);
    if (T != DSQG_F16 && small) sv.shrink();
    if (edge(t) && sv.clean()) odd[t & 1] = t + 1;
    sv.store(lds[t & 1][1]);
  };

  Acc<T, D> o;
#pragma unroll
  for (int d = 0; d < X::DB; ++d) o[d] = zero_tile();
  float m = -INFINITY, sum = 0.f;
  bool large = false;
  // The largest weight is 2^lift: float16 weights far below it stay clear of the type's subnormal numbers.
  constexpr float lift = T == DSQG_F16 ? 14.f : 0.f;
  const float far = p.scale2 < 0.f ? INFINITY : -INFINITY;  // a score of weight zero (scale2 is never zero)

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
    const char* const kt = lds[t & 1][0];
    const char* const vt = lds[t & 1][1];
    // Of a block of 32 keys the wave's queries see nothing / all.
    auto none = [&](int k0) { return k0 > i0 + 31 || (k0 + 32 <= i0 - p.window + 1 && k0 >= p.sinks); };
    auto all = [&](int k0) { return k0 + 31 <= i0 && (i0 + 31 - k0 < p.window || k0 + 32 <= p.sinks); };
    // All blocks' scores first: the matrix instructions work on the second while the first is weighed.  (Not at D = 32, where
    // four workgroups a CU do that, with 128 registers a wave.)
    constexpr bool FIRST = D > 32;
    f32x16_t x[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      if (FIRST && !none(j0 + 32 * kb)) x[kb] = scores<T, D>(kt + 32 * kb * X::RB, l, q);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int k0 = j0 + 32 * kb;
      if (none(k0)) continue;
      if (!FIRST) x[kb] = scores<T, D>(kt + 32 * kb * X::RB, l, q);
      float s[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = x[kb][r];
      const Seen seen = {i - p.window + 1 - k0, i - k0, p.sinks - k0};
      if (!all(k0)) {
        float no[1];
        hide<T>(far, seen, k0 < p.sinks, h, s, no);
      }
      float mx = s[0];
      if (p.scale2 < 0.f) {
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fminf(mx, s[r]);
      } else {
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
      }
      mx = xor32_pair_max(reference_exponent<T>(mx, p.scale2, lift));
      if (__any(mx > m)) {
        const float mn = fmaxf(m, mx), a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        large = __any(fabsf(mn) >= kLarge && mn != -INFINITY);
        sum *= a;
#pragma unroll
        for (int d = 0; d < X::DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= a;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      exponents(s, p.scale2, large, [&](int) { return ref; });
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r]);
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += s[r];
      Weights<T> f;
      pack<T>(s, f);
      contract<T, D>(o, vt + 32 * kb * X::RB, l, f);
      if (odd[t & 1] == t + 1) add_odd<T, D>(o, vh + k0 * p.v.n, p.v.n, length - k0, l, seen);
    }
    if (t + 1 < span.n) {
      store(t + 1);
      if (t + 2 < span.n) load(t + 2);
    }
    __syncthreads();
  }

  if (T != DSQG_F16 && !small) {
    float any = 0.f;
#pragma unroll
    for (int d = 0; d < X::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (D % 32 == 0 || 32 * d + 8 * (r / 4) < D) any = __builtin_fmaf(o[d][r], 0.f, any);
    if (any != any) over = 1;
    __syncthreads();
    if (over) return true;
  }
  sum = xor32_pair_sum(sum);
  const bool live = i < length && sum != 0.f;
  store_columns<T, D>(o, (small ? 0x1p30f : 1.f) / sum, live, bytes + wave * out_block<T, D>(),
                      p.out.at + b * p.out.b + head * p.out.h + i0 * p.out.n, p.out.n, p.N - i0, l);
  if constexpr (T != DSQG_F32)
    if (p.low.at)
      store_columns<T, D, true>(o, (small ? 0x1p30f : 1.f) / sum, live, bytes + wave * out_block<T, D>(),
                                p.low.at + b * p.low.b + head * p.low.h + i0 * p.low.n, p.low.n, p.N - i0, l);
  if (p.stats && h == 0 && i < p.N)
    p.stats[((long long)b * p.Hkv * p.G + head) * p.N + i] = live ? make_float2(m, 1.f / sum) : make_float2(INFINITY, 0.f);
  return false;
}

// Sums of values near the type's largest may pass it where their mean does not.  A workgroup with such a sum (or one that sees an
// infinity) goes over its tiles once more with values times 2^-30, so that sums of 2^30 rows are finite.
template <int T, int D, int NW>
__global__ __launch_bounds__(64 * NW, D <= 32 ? 4 : 2) void window_fwd_kernel(WindowParams p) {
  if constexpr (T == DSQG_F16) {  // (2^30 of its largest, times 2^14, are far from float32's)
    window_fwd_pass<T, D, NW>(p, blockIdx.x, threadIdx.x, false);
    return;
  }
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int workgroup = blockIdx.x;
    asm volatile("" : "+s"(workgroup));  // (a second pass finds its places anew: kept, they would take registers)
    if (!window_fwd_pass<T, D, NW>(p, workgroup, threadIdx.x, pass == 1)) break;
  }
}

template <int T, int D, int NW>
hipError_t launch_waves(const WindowParams& p, hipStream_t st) {
  hipLaunchKernelGGL((window_fwd_kernel<T, D, NW>), dim3((unsigned)((long long)p.B * p.Hkv * p.G * p.blocks)), dim3(64 * NW), 0, st, p);
  return hipGetLastError();
}

template <int T, int D>
hipError_t launch(const WindowParams& p, hipStream_t st) {
  if constexpr (may_be_wide(T, D))
    if (p.waves == 8) return launch_waves<T, D, 8>(p, st);
  return launch_waves<T, D, 4>(p, st);
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

hipError_t launch_window_fwd(const WindowParams& p, int dtype, hipStream_t st) {
  if (dtype == DSQG_F32) return launch_dim<DSQG_F32>(p, st);
  if (dtype == DSQG_BF16) return launch_dim<DSQG_BF16>(p, st);
  return launch_dim<DSQG_F16>(p, st);
}

}  // namespace dsqg
