// A token of each row of logits by one uniform number (gfx950): temperature, top-k, top-p, min-p, inverse CDF.
//
//   w_i = exp((x_i - max x) / T)
//
// The limits keep a first part of the order (x descending, of equal ones the lower index first): the first top_k,
// of those the ones with at most top_p of their mass before them, of those the ones with w >= min_p.  The token is the
// first, by index, whose running mass is above u times the kept mass.  So no sort is needed: the last element
// kept is found by value, and the draw is a running sum in the order of memory.
//
// Masses are whole numbers, w 2^F rounded (2^F times the row's length stays below 2^62): sums of them are exact, and so
// the same in any order.  w comes from a polynomial in 64 bits, for the sums decide between neighbours: with weights in
// fp32 one row in a few thousand of a flat distribution takes the neighbour of the token that the exact sums give.
// An element below 2^-(F+1) has no mass and is never drawn.
//
// Searching the last kept element: a histogram (counts and masses) over 2048 bins of equal width in log w; the bin
// that it lies in is searched again over its elements' bits, from a list in LDS where they are not too many, until one
// value is left.  Of m elements of that value to keep, the first m by index are found on the way of the last sum.
#include "../../include/dsqg.h"
#include "dsqg_common.hpp"

namespace dsqg {
namespace {

typedef unsigned long long u64;

struct Sample {
  const char* x; long long xs;  // logits and the bytes from row to row
  int V, F;
  const void* u; int u64bits;
  double temperature, top_p, min_p;
  long long top_k;
  const float* temperatures;    // of each row, or null
  const long long* top_ks;
  const float* top_ps;
  const float* min_ps;
  long long* out;
  float* logp;                  // or null
};

constexpr int kThreads = 1024, kW = kThreads / 64;
constexpr int kBins = 2048;   // two a thread
constexpr int kList = 4096;
constexpr int kCells = 2048;  // stretches of a row for the last sum, two a thread

template <int DT> struct Elem;
template <> struct Elem<DSQG_F32> { static constexpr int vec = 4; };
template <> struct Elem<DSQG_BF16> { static constexpr int vec = 8; };
template <> struct Elem<DSQG_F16> { static constexpr int vec = 8; };

// 16 bytes of logits as floats; a NaN is no candidate (-inf), and zeros have one sign.
template <int DT>
__device__ __forceinline__ void unpack(uint4 r, float (&x)[Elem<DT>::vec]) {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < Elem<DT>::vec; ++i) {
    float f;
    if constexpr (DT == DSQG_F32) f = __uint_as_float(w[i]);
    else if constexpr (DT == DSQG_BF16) f = __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else f = (float)__builtin_bit_cast(f16x8, r)[i];
    x[i] = f == f ? f + 0.f : -INFINITY;
  }
}

// Order of floats as that of whole numbers.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// 2^t 2^F for t <= 0 (0 below 2^-(F+2)): Taylor's series of 2^f, |f| <= 1/2, whose thirteenth term is below 2^-52.
__device__ __forceinline__ double mass_of(double t, int F) {
  if (!(t > -(double)(F + 2))) return 0.0;
  const double n = __builtin_rint(t), f = t - n;
  double p = 2.5678435993488196e-11;
  p = __builtin_fma(p, f, 4.44553827187081e-10);
  p = __builtin_fma(p, f, 7.054911620801121e-09);
  p = __builtin_fma(p, f, 1.0178086009239696e-07);
  p = __builtin_fma(p, f, 1.3215486790144305e-06);
  p = __builtin_fma(p, f, 1.5252733804059838e-05);
  p = __builtin_fma(p, f, 0.00015403530393381606);
  p = __builtin_fma(p, f, 0.0013333558146428441);
  p = __builtin_fma(p, f, 0.009618129107628477);
  p = __builtin_fma(p, f, 0.055504108664821576);
  p = __builtin_fma(p, f, 0.2402265069591007);
  p = __builtin_fma(p, f, 0.6931471805599453);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n + F);
}

// A mass (at most 2^48) as a whole number.
__device__ __forceinline__ u64 whole(double m) { return (u64)__double_as_longlong(m + 0x1p52) & 0xfffffffffffffull; }

// A row's settings and what its passes share.
struct Row {
  const char* at;  // the row from the 16-byte boundary at or before its start
  int h, V, nvec;  // elements between the two, candidates, 16-byte pieces
  int F;
  float M;         // largest logit
  double c;        // log2(e) / T
  __device__ __forceinline__ double log2_weight(float x) const { return x == M ? 0.0 : ((double)x - (double)M) * c; }
  __device__ __forceinline__ double mass(float x) const { return x == -INFINITY ? 0.0 : mass_of(log2_weight(x), F); }
  // Bins of equal width in log w, from the largest.
  __device__ __forceinline__ int bin(float x) const {
    return min(kBins - 1, (int)(-log2_weight(x) * ((double)kBins / (F + 2))));
  }
};

template <int DT, typename Fn>
__device__ __forceinline__ void piece(const Row& r, int v, Fn&& fn) {
  constexpr int VEC = Elem<DT>::vec;
  float x[VEC];
  unpack<DT>(ld16(r.at + 16ll * v), x);
  const int i0 = v * VEC - r.h;
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if ((unsigned)(i0 + e) < (unsigned)r.V) fn(x[e], i0 + e);
}

template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

struct Shared {
  uint32_t cnt[kBins];
  u64 mass[kBins];
  union {
    uint32_t lkey[kList];
    u64 cell_mass[kCells];
  };
  uint32_t cell_ties[kCells];
  u64 wm[kW];
  uint32_t wc[kW];
  uint32_t a, b, n, bin;
  u64 base;
};

// Exclusive sums over the threads' (m, c), and the totals.
__device__ __forceinline__ void block_scan(Shared& s, u64 m, uint32_t c, u64* bm, uint32_t* bc, u64* tm, uint32_t* tc) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 im = m;
  uint32_t ic = c;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 x = __shfl_up(im, o, 64);
    const uint32_t y = __shfl_up(ic, o, 64);
    if (lane >= o) { im += x; ic += y; }
  }
  __syncthreads();
  if (lane == 63) { s.wm[wave] = im; s.wc[wave] = ic; }
  __syncthreads();
  u64 pm = 0, am = 0;
  uint32_t pc = 0, ac = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    if (w == wave) { pm = am; pc = ac; }
    am += s.wm[w];
    ac += s.wc[w];
  }
  *bm = pm + im - m;
  *bc = pc + ic - c;
  *tm = am;
  *tc = ac;
}

// The last element that a limit keeps: all above `key` and the first `ties` (by index) of that value.
struct Cut {
  uint32_t key;
  uint32_t ties;
  u64 kept;  // the mass that stays
};

// One histogram, already in s.cnt and s.mass: the bin of the last element kept.  By count the limit-th element, by mass
// the last one with at most `limit` before it.  Returns false where all elements stay.
__device__ __forceinline__ bool crossing(Shared& s, bool by_mass, u64 limit, u64& base_m, uint32_t& base_c, int* bin, u64* total) {
  const int t = threadIdx.x;
  const u64 m0 = s.mass[2 * t], m1 = s.mass[2 * t + 1];
  const uint32_t c0 = s.cnt[2 * t], c1 = s.cnt[2 * t + 1];
  u64 bm, tm;
  uint32_t bc, tc;
  block_scan(s, m0 + m1, c0 + c1, &bm, &bc, &tm, &tc);
  if (t == 0) s.bin = kBins;
  __syncthreads();
  bm += base_m;
  bc += base_c;
  *total = tm + base_m;
  auto test = [&](int b, u64 m, uint32_t c, u64 before_m, uint32_t before_c) {
    if (c == 0) return;
    // By mass: the last element there is that may stay; the bin is the last whose first element does.
    const bool here = by_mass ? before_m <= limit && before_m + m > limit : before_c < limit && before_c + c >= limit;
    if (here) {
      s.bin = b;
      s.base = before_m;
      s.a = before_c;
    }
  };
  test(2 * t, m0, c0, bm, bc);
  test(2 * t + 1, m1, c1, bm + m0, bc + c0);
  __syncthreads();
  *bin = s.bin;
  if (s.bin == kBins) return false;
  base_m = s.base;
  base_c = s.a;
  __syncthreads();
  return true;
}

template <typename Each>
__device__ __forceinline__ void histogram(Shared& s, Each&& each) {
  const int t = threadIdx.x;
  __syncthreads();
  for (int b = t; b < kBins; b += kThreads) {
    s.cnt[b] = 0;
    s.mass[b] = 0;
  }
  __syncthreads();
  each([&](int b, u64 m) {
    atomicAdd(&s.cnt[b], 1u);
    atomicAdd(&s.mass[b], m);
  });
  __syncthreads();
}

// The cut inside bin `b1` of the first histogram, of which base_m and base_c lie before.
template <int DT>
__device__ Cut search(Shared& s, const Row& r, int b1, bool by_mass, u64 limit, u64 base_m, uint32_t base_c) {
  const int t = threadIdx.x;
  auto row = [&](auto&& fn) {
    for (int v = t; v < r.nvec; v += kThreads)
      piece<DT>(r, v, [&](float x, int) {
        const u64 m = whole(r.mass(x));
        if (m && r.bin(x) == b1) fn(key_of(x), m);
      });
  };
  __syncthreads();
  if (t == 0) {
    s.n = 0;
    s.a = 0xffffffffu;
    s.b = 0;
  }
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0;
  row([&](uint32_t k, u64) {
    lo = min(lo, k);
    hi = max(hi, k);
    const uint32_t at = atomicAdd(&s.n, 1u);
    if (at < kList) s.lkey[at] = k;
  });
  atomicMin(&s.a, lo);
  atomicMax(&s.b, hi);
  __syncthreads();
  lo = s.a;
  hi = s.b;
  const uint32_t n = s.n;
  auto each = [&](auto&& fn) {
    if (n <= kList) {
      for (uint32_t i = t; i < n; i += kThreads) {
        const uint32_t k = s.lkey[i];
        if (k >= lo && k <= hi) fn(k, whole(r.mass(value_of(k))));
      }
    } else {
      row([&](uint32_t k, u64 m) {
        if (k >= lo && k <= hi) fn(k, m);
      });
    }
  };
  while (lo < hi) {
    // Sub-bins of 2^shift keys from the largest down.
    const int bits = 32 - __builtin_clz(hi - lo), shift = max(0, bits - 11);
    histogram(s, [&](auto&& add) { each([&](uint32_t k, u64 m) { add((hi - k) >> shift, m); }); });
    int b;
    u64 total;
    if (!crossing(s, by_mass, limit, base_m, base_c, &b, &total)) break;  // (does not happen: the bin holds it)
    const uint32_t top = hi - ((uint32_t)b << shift);
    hi = top;
    lo = max(lo, shift == 0 ? top : top - ((1u << shift) - 1u) > top ? 0u : top - ((1u << shift) - 1u));
    if (shift == 0) break;
  }
  lo = hi;
  const u64 m = whole(r.mass(value_of(hi)));
  Cut c;
  c.key = hi;
  c.ties = by_mass ? (uint32_t)min((limit - base_m) / m + 1, (u64)0xffffffffu) : (uint32_t)(limit - base_c);
  c.kept = base_m + (u64)c.ties * m;
  __syncthreads();
  return c;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(Sample p) {
  constexpr int VEC = Elem<DT>::vec, ES = 16 / VEC;
  __shared__ Shared s;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const long long b = blockIdx.x;
  const double T = p.temperatures ? (double)p.temperatures[b] : p.temperature;
  const double top_p = p.top_ps ? (double)p.top_ps[b] : p.top_p;
  const double min_p = p.min_ps ? (double)p.min_ps[b] : p.min_p;
  const long long top_k = p.top_ks ? p.top_ks[b] : p.top_k;
  const double u = p.u64bits ? static_cast<const double*>(p.u)[b] : (double)static_cast<const float*>(p.u)[b];
  Row r;
  const unsigned long long addr = reinterpret_cast<unsigned long long>(p.x + b * p.xs);
  r.at = reinterpret_cast<const char*>(addr & ~15ull);
  r.h = (int)(addr & 15u) / ES;
  r.V = p.V;
  r.nvec = (int)(((long long)r.h + p.V + VEC - 1) / VEC);
  r.F = p.F;

  // The largest logit.
  float mx = -INFINITY;
  for (int v = t; v < r.nvec; v += kThreads) piece<DT>(r, v, [&](float x, int) { mx = fmaxf(mx, x); });
#pragma unroll
  for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if (lane == 0) s.wc[wave] = __float_as_uint(mx);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kW; ++w) mx = fmaxf(mx, __uint_as_float(s.wc[w]));
  r.M = mx;
  const bool greedy = !(T > 0.0);
  r.c = greedy ? 0.0 : 1.4426950408889634 / T;
  if (mx == -INFINITY) {  // no candidate
    if (t == 0) {
      p.out[b] = -1;
      if (p.logp) p.logp[b] = -INFINITY;
    }
    return;
  }
  __syncthreads();

  Cut cut{0u, 0u, 0};  // (all stay: no value has the key 0, which a NaN would)
  if (greedy) {
    cut = Cut{key_of(mx), 1u, 1};
  } else if ((top_k > 0 && top_k < p.V) || top_p < 1.0) {
    histogram(s, [&](auto&& add) {
      for (int v = t; v < r.nvec; v += kThreads)
        piece<DT>(r, v, [&](float x, int) {
          const u64 m = whole(r.mass(x));
          if (m) add(r.bin(x), m);
        });
    });
    u64 total = 0, bm = 0;
    uint32_t bc = 0;
    int bin;
    const bool by_count = top_k > 0 && top_k < p.V;
    bool some = crossing(s, false, by_count ? (u64)top_k : ~0ull, bm, bc, &bin, &total);
    if (by_count && some) {
      // (The first histogram is needed again for the mass.)
      u64 km[2] = {s.mass[2 * t], s.mass[2 * t + 1]};
      uint32_t kc[2] = {s.cnt[2 * t], s.cnt[2 * t + 1]};
      cut = search<DT>(s, r, bin, false, (u64)top_k, bm, bc);
      total = cut.kept;
      s.mass[2 * t] = km[0]; s.mass[2 * t + 1] = km[1];
      s.cnt[2 * t] = kc[0]; s.cnt[2 * t + 1] = kc[1];
      __syncthreads();
    }
    if (top_p < 1.0) {
      const double lim = top_p > 0.0 ? top_p * (double)total : 0.0;
      const u64 limit = min((u64)lim, total - 1);
      u64 all;
      bm = 0;
      bc = 0;
      if (crossing(s, true, limit, bm, bc, &bin, &all)) cut = search<DT>(s, r, bin, true, limit, bm, bc);
    }
  }

  // Masses of stretches of the row, in its order; tied elements are counted, for how many of them stay is known only
  // behind the sum over the stretches before.
  const double floor_mass = (min_p > 0.0 ? fmin(min_p, 1.0) : 0.0) * __builtin_amdgcn_ldexp(1.0, p.F);
  auto mass = [&](float x) -> u64 {
    const double m = r.mass(x);
    return m >= floor_mass ? whole(m) : 0;
  };
  const u64 tie_mass = cut.key ? (greedy ? 1 : mass(value_of(cut.key))) : 0;
  const int per = (int)(((long long)r.nvec + 64ll * kCells - 1) / (64ll * kCells)) * 64;  // pieces of a stretch
  const int cells = (r.nvec + per - 1) / per;
  for (int c = t; c < kCells; c += kThreads) {
    s.cell_mass[c] = 0;
    s.cell_ties[c] = 0;
  }
  __syncthreads();
  for (int c = wave; c < cells; c += kW) {
    u64 m = 0;
    uint32_t ties = 0;
    for (int v = c * per + lane; v < min((c + 1) * per, r.nvec); v += 64)
      piece<DT>(r, v, [&](float x, int) {
        const uint32_t k = key_of(x);
        if (k == cut.key) ++ties;
        else if (k > cut.key && !greedy) m += mass(x);
      });
    m = wave_sum(m);
    ties = wave_sum(ties);
    if (lane == 0) {
      s.cell_mass[c] = m;
      s.cell_ties[c] = ties;
    }
  }
  __syncthreads();
  // Sums before each stretch: ties first, which say how many of a stretch's stay.
  u64 m0 = s.cell_mass[2 * t], m1 = s.cell_mass[2 * t + 1], bm, total;
  const uint32_t c0 = s.cell_ties[2 * t], c1 = s.cell_ties[2 * t + 1];
  uint32_t bc, tc;
  block_scan(s, m0 + m1, c0 + c1, &bm, &bc, &total, &tc);
  auto stay = [&](uint32_t before, uint32_t n) { return before >= cut.ties ? 0u : min(cut.ties - before, n); };
  bm += (u64)min(bc, cut.ties) * tie_mass;
  total += (u64)min(tc, cut.ties) * tie_mass;
  m0 += (u64)stay(bc, c0) * tie_mass;
  m1 += (u64)stay(bc + c0, c1) * tie_mass;
  // (A u that is no number, or below 0, is 0; one from 1 on takes the last.)
  const double want = u > 0.0 ? u * (double)total : 0.0;
  const u64 target = want >= (double)total ? total - 1 : min((u64)want, total - 1);
  if (bm <= target && target < bm + m0) {
    s.bin = 2 * t;
    s.base = bm;
    s.a = bc;
  } else if (bm + m0 <= target && target < bm + m0 + m1) {
    s.bin = 2 * t + 1;
    s.base = bm + m0;
    s.a = bc + c0;
  }
  __syncthreads();
  if (wave != 0) return;
  // The stretch that holds the token, 64 pieces at a time.
  const int cell = s.bin;
  u64 run = s.base;
  uint32_t ties = s.a;
  for (int v0 = cell * per; v0 < min((cell + 1) * per, r.nvec); v0 += 64) {
    const int v = v0 + lane;
    u64 m = 0;
    uint32_t n = 0;
    if (v < r.nvec)
      piece<DT>(r, v, [&](float x, int) {
        const uint32_t k = key_of(x);
        if (k == cut.key) ++n;
        else if (k > cut.key && !greedy) m += mass(x);
      });
    uint32_t tn = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(tn, o, 64);
      if (lane >= o) tn += y;
    }
    const uint32_t before = ties + tn - n;
    m += (u64)stay(before, n) * tie_mass;
    u64 im = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 y = __shfl_up(im, o, 64);
      if (lane >= o) im += y;
    }
    const u64 first = run + im - m;
    if (first <= target && target < first + m) {
      u64 at = first;
      uint32_t tb = before;
      bool done = false;
      piece<DT>(r, v, [&](float x, int i) {
        const uint32_t k = key_of(x);
        u64 w = 0;
        if (k == cut.key) w = tb++ < cut.ties ? tie_mass : 0;
        else if (k > cut.key && !greedy) w = mass(x);
        at += w;
        if (!done && at > target) {
          done = true;
          p.out[b] = i;
          // log(w / K) = (x - M) / T - log K.
          if (p.logp) {
            const double lw = r.log2_weight(x) * 0.6931471805599453;
            p.logp[b] = greedy ? 0.f : (float)(lw - log((double)total * __builtin_amdgcn_ldexp(1.0, -p.F)));
          }
        }
      });
    }
    run += __shfl(im, 63, 64);
    ties += __shfl(tn, 63, 64);
    if (run > target) break;
  }
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" int dsqg_sample(const dsqg_sample_args* a, dsqg_stream_t stream) {
  if (!a || a->B < 0 || a->V < 1) return DSQG_EINVAL;
  if (a->dtype != DSQG_F32 && a->dtype != DSQG_BF16 && a->dtype != DSQG_F16) return DSQG_EINVAL;
  if (a->B == 0) return DSQG_OK;
  if (!a->logits || !a->u || !a->tokens) return DSQG_EINVAL;
  const long long es = a->dtype == DSQG_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->logits) % es != 0 || a->logits_stride < 0 || a->logits_stride > (1ll << 50)) return DSQG_EINVAL;
  if (a->V > (1 << 30)) return DSQG_EUNSUPPORTED;
  if (a->u_is_double != 0 && a->u_is_double != 1) return DSQG_EINVAL;
  // (A setting that is not a number keeps nothing out: refused here, an off switch where rows have their own.)
  if (a->temperature != a->temperature || a->top_p != a->top_p || a->min_p != a->min_p) return DSQG_EINVAL;
  Sample p = {};
  p.x = static_cast<const char*>(a->logits);
  p.xs = a->logits_stride * es;
  p.V = a->V;
  int bits = 0;
  while ((1ll << bits) < a->V) ++bits;
  p.F = bits > 14 ? 62 - bits : 48;
  p.u = a->u;
  p.u64bits = a->u_is_double;
  p.temperature = a->temperature;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.top_k = a->top_k;
  p.temperatures = a->temperatures;
  p.top_ks = reinterpret_cast<const long long*>(a->top_ks);
  p.top_ps = a->top_ps;
  p.min_ps = a->min_ps;
  p.out = reinterpret_cast<long long*>(a->tokens);
  p.logp = a->logprobs;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)a->B), block(kThreads);
  if (a->dtype == DSQG_F32) hipLaunchKernelGGL(sample_kernel<DSQG_F32>, grid, block, 0, st, p);
  else if (a->dtype == DSQG_BF16) hipLaunchKernelGGL(sample_kernel<DSQG_BF16>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(sample_kernel<DSQG_F16>, grid, block, 0, st, p);
  return hipGetLastError() == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
