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
// Searching the last kept element: 2048 bins of equal width in log w.  With top-k the bin below which nothing counts is that
// of the k-th largest of many stretches' maxima, and what lies above it, little more than k elements, is put into a list;
// with top-p alone the bin comes from a histogram of masses, and its elements are the list.  The list is sorted.  A row whose
// list is too long (nearly equal logits, a top-k of thousands) goes the general way, by histograms of histograms.
//
// A row takes one workgroup where there are rows for all CUs; fewer rows are split, each over up to eight, and four launches
// take the place of the barriers between the steps.  (256 rows of 32000 bfloat16 in two parts each: 65 us, in one 39.)
//
// Measured: 1 row of 32000 float32, top-p, 25 us in its four launches (one workgroup: 72); 256 rows of 32000 bfloat16 with top-k,
// top-p and temperatures of their own, 39 us; 64 rows of 151001 float32, top-p and min-p, 62 us, of which the masses take 43: two
// passes of some 40 vector instructions an element, half of them in 64 bits.  Memory would take 3 and 8 us; a
// single row's launches wait for memory and for each other.
#include <algorithm>

#include "../../include/dsqg.h"
#include "dsqg_common.hpp"

namespace dsqg {
namespace {

typedef unsigned long long u64;

struct Sample {
  const char* x; long long xs;  // logits and the bytes from row to row
  int V, bits, F;               // ... ceil(log2 V), a whole mass's bits
  const void* u; int u64bits;
  double temperature, top_p, min_p;
  long long top_k;
  const float* temperatures;    // of each row, or null
  const long long* top_ks;
  const float* top_ps;
  const float* min_ps;
  long long* out;
  float* logp;                  // or null
  // Rows split over S workgroups: what these leave for the next launch.
  int S;
  float* maxima;                // [B, S, kThreads]
  u64* mass;                    // [B, S, kBins]
  u64* list;                    // [B, S, kList]
  u64* cells;                   // [B, kCells]
  uint32_t* counts;             // [B, S]: lengths of the lists
  u64* found;                   // [B, 3]: the largest logit, the mass before the list, the mass of all
};

constexpr int kThreads = 1024, kW = kThreads / 64;
constexpr int kBins = 2048;   // two a thread
constexpr int kList = 4096;
constexpr int kCells = 2048;  // stretches of a row for the last sum, two a thread
constexpr int kSplit = 8;     // workgroups of a row, at most
constexpr int kTop = 1024;     // largest top-k by maxima: half of a workgroup's

// A row is taken in pieces of four elements, 16 or 8 bytes.
constexpr int kVec = 4;
template <int DT> struct Elem { typedef uint2 raw; static constexpr int size = 2; };
template <> struct Elem<DSQG_F32> { typedef uint4 raw; static constexpr int size = 4; };
template <int DT> using Raw = typename Elem<DT>::raw;

// A NaN is no candidate: -inf.
template <int DT>
__device__ __forceinline__ void unpack(Raw<DT> r, float (&x)[kVec]) {
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    float f;
    if constexpr (DT == DSQG_F32) {
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
      f = __uint_as_float(w[i]);
    } else if constexpr (DT == DSQG_BF16) {
      const uint32_t w[2] = {r.x, r.y};
      f = __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    } else {
      f = (float)__builtin_bit_cast(f16x4, r)[i];
    }
    x[i] = fmaxf(f, -INFINITY);
  }
}

// Order of floats as that of whole numbers.  (Zeros have one sign.)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// 2^t 2^F for t <= 0, whole(..) of which is 0 below 2^-(F+1), and for what is no number: Taylor's series of 2^f, |f| <= 1/2, whose
// thirteenth term is below 2^-52.  The addition of 1.5 2^52 + F rounds t and leaves its whole part plus F in the low bits.
__device__ __forceinline__ double mass_of(double t, int F) {
  const double magic = 0x1.8p52 + F;
  t = fmax(t, -(double)(F + 2));
  const double s = t + magic, f = t - (s - magic);
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
  return __builtin_amdgcn_ldexp(p, (int)(uint32_t)__double_as_longlong(s));
}

// A mass (at most 2^48) as a whole number.
__device__ __forceinline__ u64 whole(double m) { return (u64)__double_as_longlong(m + 0x1p52) & 0xfffffffffffffull; }

// A row's settings and what its passes share.
struct Row {
  const char* at;  // the row from the first piece's boundary at or before its start
  int h, V, nvec;  // elements between the two, candidates, pieces
  int F;
  float M;         // largest logit
  double c;        // log2(e) / T
  float bins;      // bins of a unit of x
  int per, cells;  // pieces of a stretch (64 or a multiple), and stretches
  __device__ __forceinline__ double log2_weight(float x) const { return x == M ? 0.0 : ((double)x - (double)M) * c; }
  // Whether differences and their products are numbers; else the general way goes by mass_any.
  __device__ __forceinline__ bool usual() const { return M < INFINITY && c < __builtin_huge_val() && bins < INFINITY && bins > 0.f; }
  __device__ __forceinline__ double mass(float x) const { return mass_of(((double)x - (double)M) * c, F); }
  __device__ __forceinline__ double mass_any(float x) const { return x == -INFINITY ? 0.0 : mass_of(log2_weight(x), F); }
  // Bins of equal width in log w, from the largest.  (Each step's rounding keeps the order.)
  __device__ __forceinline__ int bin(float x) const { return (int)fminf((M - x) * bins, (float)(kBins - 1)); }
  __device__ __forceinline__ int bin_any(float x) const { return x == M ? 0 : bin(x); }
  // Elements in order: the larger first, of equal ones the lower index.
  __device__ __forceinline__ static u64 rank(float x, int i) { return (u64)key_of(x) << 32 | ~(uint32_t)i; }
  __device__ __forceinline__ int cell(int i) const { return (i + h) / kVec / per; }
};

template <int DT>
__device__ __forceinline__ Raw<DT> load(const Row& r, int v) {
  return *reinterpret_cast<const Raw<DT>*>(r.at + (long long)sizeof(Raw<DT>) * min(v, r.nvec - 1));
}

template <int DT>
__device__ __forceinline__ float element(const Row& r, int i) {
  float x[kVec];
  Raw<DT> raw = {};
  const char* const at = r.at + (long long)(i + r.h) * Elem<DT>::size;
  if constexpr (DT == DSQG_F32) raw.x = *reinterpret_cast<const uint32_t*>(at);
  else raw.x = *reinterpret_cast<const unsigned short*>(at);
  unpack<DT>(raw, x);
  return x[0];
}

// fn(x, index) of the elements of a lane's piece, those of a wave following each other.  Elements outside the row have no weight.
template <int DT, typename Fn>
__device__ __forceinline__ void piece(const Row& r, int v, Raw<DT> raw, Fn&& fn) {
  float x[kVec];
  unpack<DT>(raw, x);
  const int i0 = v * kVec - r.h, wave0 = __builtin_amdgcn_readfirstlane(i0 - (int)(threadIdx.x & 63) * kVec);
  if (wave0 < 0 || wave0 + 64 * kVec > r.V) {
    asm volatile("");  // (a branch of the row's ends)
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if ((unsigned)(i0 + e) >= (unsigned)r.V) x[e] = -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) fn(x[e], i0 + e);
}

// fn(piece, its data) for a workgroup's pieces v0 .. v1, whole waves at a time (64 pieces from a multiple of 64 on); the next
// one is on its way meanwhile.
template <int DT, typename Fn>
__device__ __forceinline__ void pieces(const Row& r, int v0, int v1, Fn&& fn) {
  int v = v0 + (int)threadIdx.x;
  Raw<DT> next = load<DT>(r, v);
#pragma unroll 1
  for (; v - (int)(threadIdx.x & 63) < v1; v += kThreads) {
    const Raw<DT> raw = next;
    next = load<DT>(r, v + kThreads);
    fn(v, raw);
  }
}

template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xf, true);
  return (u64)hi << 32 | lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, true);
}

// Sums over the lanes up to each (of each row of 16, where N is 16).  All lanes take part.
template <int N = 64, typename T>
__device__ __forceinline__ T wave_scan(T x) {
  x += moved<0x111, 0xf>(x);
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  if constexpr (N == 64) {
    x += moved<0x142, 0xa>(x);
    x += moved<0x143, 0xc>(x);
  }
  return x;
}

__device__ __forceinline__ u64 lane_of(u64 x, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

struct Shared {
  uint32_t cnt[kBins];
  u64 mass[kBins];
  union {
    u64 list[kList];
    struct {  // the general way
      uint32_t lkey[kList];
      uint32_t cell_ties[kCells];
    };
  };
  u64 cells[kCells];
  u64 wm[kW];
  uint32_t wc[kW];
  uint32_t a, b, n, bin;
  u64 base, cut;
  Sample p;  // for the general way
  long long b64;
  float largest;
};

// Exclusive sums over the threads' (m, c), and the totals.
__device__ __forceinline__ void block_scan(Shared& s, u64 m, uint32_t c, u64* bm, uint32_t* bc, u64* tm, uint32_t* tc) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u64 im = wave_scan(m);
  const uint32_t ic = wave_scan(c);
  __syncthreads();
  if (lane == 63) { s.wm[wave] = im; s.wc[wave] = ic; }
  __syncthreads();
  // (Each wave adds the sixteen waves' sums for itself.)
  static_assert(kW == 16, "a row of lanes");
  const u64 sm = wave_scan<16>(s.wm[lane & 15]);
  const uint32_t sc = wave_scan<16>(s.wc[lane & 15]);
  *tm = lane_of(sm, 15);
  *tc = __builtin_amdgcn_readlane(sc, 15);
  *bm = (wave ? lane_of(sm, wave - 1) : 0) + im - m;
  *bc = (wave ? (uint32_t)__builtin_amdgcn_readlane(sc, wave - 1) : 0) + ic - c;
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
      piece<DT>(r, v, load<DT>(r, v), [&](float x, int) {
        const u64 m = whole(r.mass_any(x));
        if (m && r.bin_any(x) == b1) fn(key_of(x), m);
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
        if (k >= lo && k <= hi) fn(k, whole(r.mass_any(value_of(k))));
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
  const u64 m = whole(r.mass_any(value_of(hi)));
  Cut c;
  c.key = hi;
  c.ties = by_mass ? (uint32_t)min((limit - base_m) / m + 1, (u64)0xffffffffu) : (uint32_t)(limit - base_c);
  c.kept = base_m + (u64)c.ties * m;
  __syncthreads();
  return c;
}

// The mass before the last element that top_p < 1 keeps is at most this.
__device__ __forceinline__ u64 mass_limit(double top_p, u64 total) {
  const double lim = top_p > 0.0 ? top_p * (double)total : 0.0;
  return min((u64)lim, total - 1);
}

// The mass that the draw stops behind.  (A u that is no number, or below 0, is 0; one from 1 on takes the last.)
__device__ __forceinline__ u64 drawn(double u, u64 total) {
  const double want = u > 0.0 ? u * (double)total : 0.0;
  return want >= (double)total ? total - 1 : min((u64)want, total - 1);
}

// A row's own settings.
struct Want {
  double T, u, top_p, min_p;
  long long top_k;
  bool greedy, by_count;
  double floor_mass;  // of min_p
  __device__ __forceinline__ Want(const Sample& p, long long b) {
    T = p.temperatures ? (double)p.temperatures[b] : p.temperature;
    top_p = p.top_ps ? (double)p.top_ps[b] : p.top_p;
    min_p = p.min_ps ? (double)p.min_ps[b] : p.min_p;
    top_k = p.top_ks ? p.top_ks[b] : p.top_k;
    u = p.u64bits ? static_cast<const double*>(p.u)[b] : (double)static_cast<const float*>(p.u)[b];
    greedy = !(T > 0.0);
    if (greedy) top_k = 1;
    by_count = top_k > 0 && top_k < p.V;
    floor_mass = (min_p > 0.0 ? fmin(min_p, 1.0) : 0.0) * __builtin_amdgcn_ldexp(1.0, p.F);
  }
};

template <int DT>
__device__ __forceinline__ Row row_of(const Sample& p, long long b) {
  Row r;
  // (By pointers, which the compiler knows to be global memory's; from a number it makes loads that wait for LDS too.)
  const char* const x = p.x + b * p.xs;
  const int over = (int)(reinterpret_cast<uintptr_t>(x) & (sizeof(Raw<DT>) - 1));
  r.at = x - over;
  r.h = over / Elem<DT>::size;
  r.V = p.V;
  r.nvec = (int)(((long long)r.h + p.V + kVec - 1) / kVec);
  r.F = p.F;
  r.per = (int)(((long long)r.nvec + 64ll * kCells - 1) / (64ll * kCells)) * 64;
  r.cells = (r.nvec + r.per - 1) / r.per;
  return r;
}

__device__ __forceinline__ void weigh(Row& r, const Sample& p, const Want& w, float largest) {
  r.M = largest;
  r.c = w.greedy ? 1.0 : 1.4426950408889634 / w.T;
  // As far as there is mass; with top-p alone to where all that is less makes up at most 2^-7 of the largest, in narrower bins.
  r.bins = (float)(r.c * kBins / (w.by_count ? r.F + 2 : p.bits + 7));
}

// log(w / K) = (x - M) / T - log K.
__device__ __forceinline__ void log_weight(const Sample& p, long long b, const Row& r, const Want& w, float x, u64 total) {
  if (!p.logp) return;
  const double lw = r.log2_weight(x) * 0.6931471805599453;
  p.logp[b] = w.greedy ? 0.f : (float)(lw - log((double)total * __builtin_amdgcn_ldexp(1.0, -p.F)));
}

// The general way, for any row.
template <int DT>
__device__ __attribute__((noinline)) void general(Shared& s) {
  const Sample p = s.p;
  const long long b = s.b64;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const Want w(p, b);
  Row r = row_of<DT>(p, b);
  weigh(r, p, w, s.largest);
  __syncthreads();

  Cut cut{0u, 0u, 0};  // (all stay: no value has the key 0, which a NaN would)
  if (w.greedy) {
    cut = Cut{key_of(r.M), 1u, 1};
  } else {
    histogram(s, [&](auto&& add) {
      for (int v = t; v < r.nvec; v += kThreads)
        piece<DT>(r, v, load<DT>(r, v), [&](float x, int) {
          const u64 m = whole(r.mass_any(x));
          if (m) add(r.bin_any(x), m);
        });
    });
    u64 total = 0, bm = 0;
    uint32_t bc = 0;
    int bin;
    const bool by_count = w.top_k > 0 && w.top_k < p.V;
    bool some = crossing(s, false, by_count ? (u64)w.top_k : ~0ull, bm, bc, &bin, &total);
    if (by_count && some) {
      // (The first histogram is needed again for the mass.)
      u64 km[2] = {s.mass[2 * t], s.mass[2 * t + 1]};
      uint32_t kc[2] = {s.cnt[2 * t], s.cnt[2 * t + 1]};
      cut = search<DT>(s, r, bin, false, (u64)w.top_k, bm, bc);
      total = cut.kept;
      s.mass[2 * t] = km[0]; s.mass[2 * t + 1] = km[1];
      s.cnt[2 * t] = kc[0]; s.cnt[2 * t + 1] = kc[1];
      __syncthreads();
    }
    if (w.top_p < 1.0) {
      const u64 limit = mass_limit(w.top_p, total);
      u64 all;
      bm = 0;
      bc = 0;
      if (crossing(s, true, limit, bm, bc, &bin, &all)) cut = search<DT>(s, r, bin, true, limit, bm, bc);
    }
  }

  // Masses of stretches of the row, in its order; tied elements are counted, for how many of them stay is known only
  // behind the sum over the stretches before.
  auto mass = [&](float x) -> u64 {
    const double m = r.mass_any(x);
    return m >= w.floor_mass ? whole(m) : 0;
  };
  const u64 tie_mass = cut.key ? (w.greedy ? 1 : mass(value_of(cut.key))) : 0;
  for (int c = t; c < kCells; c += kThreads) {
    s.cells[c] = 0;
    s.cell_ties[c] = 0;
  }
  __syncthreads();
  for (int c = wave; c < r.cells; c += kW) {
    u64 m = 0;
    uint32_t ties = 0;
    for (int v = c * r.per + lane; v < min((c + 1) * r.per, r.nvec); v += 64)
      piece<DT>(r, v, load<DT>(r, v), [&](float x, int) {
        const uint32_t k = key_of(x);
        if (k == cut.key) ++ties;
        else if (k > cut.key && !w.greedy) m += mass(x);
      });
    m = wave_scan(m);
    ties = wave_scan(ties);
    if (lane == 63) {
      s.cells[c] = m;
      s.cell_ties[c] = ties;
    }
  }
  __syncthreads();
  // Sums before each stretch: ties first, which say how many of a stretch's stay.
  u64 m0 = s.cells[2 * t], m1 = s.cells[2 * t + 1], bm, total;
  const uint32_t c0 = s.cell_ties[2 * t], c1 = s.cell_ties[2 * t + 1];
  uint32_t bc, tc;
  block_scan(s, m0 + m1, c0 + c1, &bm, &bc, &total, &tc);
  auto stay = [&](uint32_t before, uint32_t n) { return before >= cut.ties ? 0u : min(cut.ties - before, n); };
  bm += (u64)min(bc, cut.ties) * tie_mass;
  total += (u64)min(tc, cut.ties) * tie_mass;
  m0 += (u64)stay(bc, c0) * tie_mass;
  m1 += (u64)stay(bc + c0, c1) * tie_mass;
  const u64 target = drawn(w.u, total);
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
  for (int v0 = cell * r.per; v0 < min((cell + 1) * r.per, r.nvec); v0 += 64) {
    const int v = v0 + lane;
    u64 m = 0;
    uint32_t n = 0;
    if (v < r.nvec)
      piece<DT>(r, v, load<DT>(r, v), [&](float x, int) {
        const uint32_t k = key_of(x);
        if (k == cut.key) ++n;
        else if (k > cut.key && !w.greedy) m += mass(x);
      });
    const uint32_t tn = wave_scan(n);
    const uint32_t before = ties + tn - n;
    m += (u64)stay(before, n) * tie_mass;
    const u64 im = wave_scan(m);
    const u64 first = run + im - m;
    if (first <= target && target < first + m) {
      u64 at = first;
      uint32_t tb = before;
      bool done = false;
      piece<DT>(r, v, load<DT>(r, v), [&](float x, int i) {
        const uint32_t k = key_of(x);
        u64 mine = 0;
        if (k == cut.key) mine = tb++ < cut.ties ? tie_mass : 0;
        else if (k > cut.key && !w.greedy) mine = mass(x);
        at += mine;
        if (!done && at > target) {
          done = true;
          p.out[b] = i;
          log_weight(p, b, r, w, x, total);
        }
      });
    }
    run += __shfl(im, 63, 64);
    ties += __shfl(tn, 63, 64);
    if (run > target) break;
  }
}


// ---- A row's steps, each by a workgroup on its stretches c0 .. c1. ----

// Largest of this thread's elements: of every other piece each.
template <int DT>
__device__ __forceinline__ void maxima(const Row& r, int c0, int c1, float (&m)[2]) {
  constexpr int AHEAD = 4;
  m[0] = m[1] = -INFINITY;
  const int v1 = min(c1 * r.per, r.nvec);
#pragma unroll 1
  for (int v = c0 * r.per + (int)threadIdx.x; v < v1; v += AHEAD * kThreads) {
    Raw<DT> raw[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) raw[i] = load<DT>(r, v + i * kThreads);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (v + i * kThreads < v1) piece<DT>(r, v + i * kThreads, raw[i], [&](float x, int) { m[i & 1] = fmaxf(m[i & 1], x); });
  }
}

__device__ __forceinline__ float block_max(Shared& s, float m) {
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wc[threadIdx.x >> 6] = __float_as_uint(m);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kW; ++w) m = fmaxf(m, __uint_as_float(s.wc[w]));
  return m;
}

__device__ __forceinline__ void append(Shared& s, u64 x) {
  const uint32_t at = atomicAdd(&s.n, 1u);
  if (at < (uint32_t)kList) s.list[at] = x;
}

// The elements that may be among the first top_k: each(fn) goes over maxima of parts of the row, of which top_k are not
// below the bin found.
template <int DT, typename Each>
__device__ __forceinline__ void collect(Shared& s, const Row& r, int c0, int c1, long long top_k, Each&& each) {
  const int t = threadIdx.x;
  s.cnt[t] = s.cnt[t + kThreads] = 0;
  if (t == 0) {
    s.bin = kBins - 1;
    s.n = 0;
  }
  __syncthreads();
  each([&](float m) {
    if (m != -INFINITY) atomicAdd(&s.cnt[r.bin(m)], 1u);
  });
  __syncthreads();
  const uint32_t n0 = s.cnt[2 * t], n1 = s.cnt[2 * t + 1];
  u64 bm, tm;
  uint32_t bc, tc;
  block_scan(s, 0, n0 + n1, &bm, &bc, &tm, &tc);
  if (bc < top_k && bc + n0 >= top_k) s.bin = 2 * t;
  else if (bc + n0 < top_k && bc + n0 + n1 >= top_k) s.bin = 2 * t + 1;
  __syncthreads();
  const int last = s.bin;
  pieces<DT>(r, c0 * r.per, min(c1 * r.per, r.nvec), [&](int v, Raw<DT> raw) {
    piece<DT>(r, v, raw, [&](float x, int i) {
      const int at = r.bin(x);
      // (Elements without mass are in the last bin.)
      if (at <= last && (at < kBins - 1 || whole(r.mass(x)))) append(s, r.rank(x, i));
    });
  });
  __syncthreads();
}

// Masses of the bins, in s.mass.
template <int DT>
__device__ __forceinline__ void mass_bins(Shared& s, const Row& r, int c0, int c1) {
  const int t = threadIdx.x;
  s.mass[t] = s.mass[t + kThreads] = 0;
  __syncthreads();
  pieces<DT>(r, c0 * r.per, min(c1 * r.per, r.nvec), [&](int v, Raw<DT> raw) {
    u64 m[kVec];
    int bin[kVec], n = 0;
    piece<DT>(r, v, raw, [&](float x, int) {
      m[n] = whole(r.mass(x));
      bin[n++] = r.bin(x);
    });
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (m[e]) atomicAdd(&s.mass[bin[e]], m[e]);
  });
  __syncthreads();
}

// The bin that top_p ends in, from s.mass; the mass before it and of all.
__device__ __forceinline__ int end_bin(Shared& s, double top_p, u64* base, u64* total) {
  const int t = threadIdx.x;
  const u64 m0 = s.mass[2 * t], m1 = s.mass[2 * t + 1];
  u64 bm, tm;
  uint32_t bc, tc;
  block_scan(s, m0 + m1, 0, &bm, &bc, &tm, &tc);
  const u64 limit = mass_limit(top_p, tm);
  if (bm <= limit && bm + m0 > limit) {
    s.bin = 2 * t;
    s.base = bm;
  } else if (bm + m0 <= limit && bm + m0 + m1 > limit) {
    s.bin = 2 * t + 1;
    s.base = bm + m0;
  }
  __syncthreads();
  *base = s.base;
  *total = tm;
  return s.bin;
}

// The mass of each stretch's elements of bins before `end`, added to s.cells; those of bin `end` are listed.
template <int DT>
__device__ __forceinline__ void cell_sums(Shared& s, const Row& r, const Want& w, int c0, int c1, int end) {
  const int t = threadIdx.x, lane = t & 63;
  if (t == 0) s.n = 0;
  __syncthreads();
  pieces<DT>(r, c0 * r.per, min(c1 * r.per, r.nvec), [&](int v, Raw<DT> raw) {
    u64 m = 0;
    bool some = false;
    piece<DT>(r, v, raw, [&](float x, int) {
      const int at = r.bin(x);
      const double mine = r.mass(x);
      m += at < end && mine >= w.floor_mass ? whole(mine) : 0;
      some |= at == end;
    });
    if (some) {
      asm volatile("");  // (a branch, apart from the sums)
      piece<DT>(r, v, raw, [&](float x, int i) {
        if (r.bin(x) == end && x != -INFINITY) append(s, r.rank(x, i));
      });
    }
    m = wave_scan(m);
    if (lane == 63) atomicAdd(&s.cells[v / r.per], m);
  });
  __syncthreads();
}

// The list in order, from the largest.  Up to kThreads elements: each is put where its rank says, the number of larger
// ones, of which a wave counts a sixteenth for all elements.
__device__ __forceinline__ void sort_few(Shared& s) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, n = (int)s.n;
  s.cnt[t] = 0;
  const u64 mine = t < n ? s.list[t] : 0;
  __syncthreads();
  const int each = (n + kW - 1) / kW, j0 = wave * each, j1 = min(j0 + each, n);
  for (int i = lane; i < n; i += 64) {
    const u64 x = s.list[i];
    uint32_t above = 0;
#pragma unroll 4
    for (int j = j0; j < j1; ++j) above += s.list[j] > x ? 1u : 0u;
    if (above) atomicAdd(&s.cnt[i], above);
  }
  __syncthreads();
  if (t < n) s.list[s.cnt[t]] = mine;
  __syncthreads();
}

// Of more, by a bitonic network.
__device__ __forceinline__ void sort_many(Shared& s) {
  const int t = threadIdx.x;
  const int n = (int)s.n;
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + t; i < size; i += kThreads) s.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j; j /= 2) {
      for (int e = t; e < size / 2; e += kThreads) {
        const int i = 2 * e - (e & (j - 1));
        const u64 x = s.list[i], y = s.list[i + j];
        if ((x < y) == ((i & k) == 0)) {
          s.list[i] = y;
          s.list[i + j] = x;
        }
      }
      __syncthreads();
    }
}

// What the limits leave of the list: its elements' masses go to their stretches, the last of them is s.cut.
template <int DT, int PT>
__device__ __forceinline__ void settle(Shared& s, const Row& r, const Want& w, u64 base, u64 total) {
  const int t = threadIdx.x, n = (int)s.n;
  const int kept = w.by_count ? (int)min((long long)n, w.top_k) : n;
  u64 x[PT], m[PT], sum = 0;
  double exact[PT];
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int at = PT * t + i;
    x[i] = at < kept ? s.list[at] : 0;
    exact[i] = at < kept ? r.mass(value_of((uint32_t)(x[i] >> 32))) : 0.0;
    m[i] = whole(exact[i]);
    sum += m[i];
  }
  u64 before, all;
  uint32_t bc, tc;
  block_scan(s, sum, 0, &before, &bc, &all, &tc);
  const u64 limit = w.by_count ? (w.top_p < 1.0 ? mass_limit(w.top_p, all) : ~0ull) : mass_limit(w.top_p, total);
  before += base;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int at = PT * t + i;
    if (at < kept && before <= limit) {
      if (exact[i] >= w.floor_mass) atomicAdd(&s.cells[r.cell((int)~(uint32_t)x[i])], m[i]);
      if (at == kept - 1 || before + m[i] > limit) s.cut = x[i];
    }
    before += m[i];
  }
  __syncthreads();
}

// The draw, from the stretches' masses (of s.cells; 0 beyond the row's) and the list of those elements that a limit may cut
// between: `base` of mass before them, `total` of all (none: no limit by mass but within the list).
template <int DT>
__device__ __forceinline__ void finish(Shared& s, const Sample& p, long long b, const Row& r, const Want& w, bool listed, u64 base, u64 total) {
  const int t = threadIdx.x;
  if (t == 0) s.cut = 0;
  if (listed) {
    if (s.n <= (uint32_t)kThreads) {
      sort_few(s);
      settle<DT, 1>(s, r, w, base, total);
    } else {
      sort_many(s);
      settle<DT, kList / kThreads>(s, r, w, base, total);
    }
  }
  u64 m0 = s.cells[2 * t], m1 = s.cells[2 * t + 1], bm, sum;
  uint32_t bc, tc;
  block_scan(s, m0 + m1, 0, &bm, &bc, &sum, &tc);
  const u64 target = drawn(w.u, sum);
  if (bm <= target && target < bm + m0) {
    s.bin = 2 * t;
    s.base = bm;
  } else if (bm + m0 <= target && target < bm + m0 + m1) {
    s.bin = 2 * t + 1;
    s.base = bm + m0;
  }
  __syncthreads();
  // The stretch that holds the token, an element a thread.
  const int cell = s.bin;
  const u64 cut = s.cut;
  u64 run = s.base;
  const int i1 = min((cell + 1) * r.per * kVec - r.h, p.V);
#pragma unroll 1
  for (int i0 = cell * r.per * kVec - r.h; i0 < i1; i0 += kThreads) {
    const int i = i0 + t;
    u64 m = 0;
    float x = 0.f;
    if (i >= 0 && i < i1) {
      x = element<DT>(r, i);
      const double exact = r.mass(x);
      m = r.rank(x, i) >= cut && exact >= w.floor_mass ? whole(exact) : 0;
    }
    u64 before, all;
    block_scan(s, m, 0, &before, &bc, &all, &tc);
    before += run;
    if (before <= target && target < before + m) {
      p.out[b] = i;
      log_weight(p, b, r, w, x, sum);
    }
    run += all;
    if (run > target) break;
  }
}

// No candidate in the row: says so.
__device__ __forceinline__ bool none(const Sample& p, long long b, float largest) {
  if (largest != -INFINITY) return false;
  if (threadIdx.x == 0) {
    p.out[b] = -1;
    if (p.logp) p.logp[b] = -INFINITY;
  }
  return true;
}

template <int DT>
__device__ __forceinline__ void hand_over(Shared& s, const Sample& p, long long b, float largest) {
  __syncthreads();
  if (threadIdx.x == 0) {
    s.p = p;
    s.b64 = b;
    s.largest = largest;
  }
  __syncthreads();
  general<DT>(s);
}

// A limit by count whose elements are not collected by maxima, or weights of infinities.
__device__ __forceinline__ bool needs_general(const Row& r, const Want& w) {
  return !r.usual() || (w.by_count && w.top_k > kTop && r.V > kList);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(Sample p) {
  __shared__ Shared s;
  const int t = threadIdx.x;
  const long long b = blockIdx.x;
  const Want w(p, b);
  Row r = row_of<DT>(p, b);
  float m[2];
  maxima<DT>(r, 0, r.cells, m);
  const float largest = block_max(s, fmaxf(m[0], m[1]));
  if (none(p, b, largest)) return;
  weigh(r, p, w, largest);
  u64 base = 0, total = 0;
  const bool limits = w.by_count || w.top_p < 1.0;
  s.cells[t] = s.cells[t + kThreads] = 0;
  __syncthreads();
  bool plain = !needs_general(r, w);
  if (plain) {
    if (w.by_count) {
      collect<DT>(s, r, 0, r.cells, w.top_k, [&](auto&& fn) {
        fn(m[0]);
        fn(m[1]);
      });
    } else {
      int end = kBins;
      if (limits) {
        mass_bins<DT>(s, r, 0, r.cells);
        end = end_bin(s, w.top_p, &base, &total);
      }
      cell_sums<DT>(s, r, w, 0, r.cells, end);
    }
    plain = s.n <= (uint32_t)kList;
  }
  if (!plain) {
    hand_over<DT>(s, p, b, largest);
    return;
  }
  finish<DT>(s, p, b, r, w, limits, base, total);
}

// ---- Rows split over S workgroups. ----

struct Part {
  long long b;
  int c0, c1;
  __device__ __forceinline__ Part(const Sample& p, const Row& r, long long row, int at) {
    b = row;
    const int each = (r.cells + p.S - 1) / p.S;
    c0 = min(at * each, r.cells);
    c1 = min(c0 + each, r.cells);
  }
};

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_maxima_kernel(Sample p) {
  const long long b = blockIdx.x / p.S;
  const Row r = row_of<DT>(p, b);
  const Part part(p, r, b, blockIdx.x % p.S);
  float m[2];
  maxima<DT>(r, part.c0, part.c1, m);
  p.maxima[(long long)blockIdx.x * kThreads + threadIdx.x] = fmaxf(m[0], m[1]);
}

// With top-k the list, else the bins' masses.
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(Sample p) {
  __shared__ Shared s;
  const int t = threadIdx.x;
  const long long b = blockIdx.x / p.S;
  const Want w(p, b);
  Row r = row_of<DT>(p, b);
  const Part part(p, r, b, blockIdx.x % p.S);
  float m[kSplit], largest = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSplit; ++i) {
    m[i] = i < p.S ? p.maxima[(b * p.S + i) * kThreads + t] : -INFINITY;
    largest = fmaxf(largest, m[i]);
  }
  largest = block_max(s, largest);
  if (t == 0 && blockIdx.x % p.S == 0) p.found[3 * b] = __float_as_uint(largest);
  if (largest == -INFINITY) return;
  weigh(r, p, w, largest);
  if (needs_general(r, w)) return;
  if (w.by_count) {
    collect<DT>(s, r, part.c0, part.c1, w.top_k, [&](auto&& fn) {
#pragma unroll
      for (int i = 0; i < kSplit; ++i) fn(m[i]);
    });
    const uint32_t n = s.n;
    if (t == 0) p.counts[blockIdx.x] = n;
    for (uint32_t i = t; i < min(n, (uint32_t)kList); i += kThreads) p.list[(long long)blockIdx.x * kList + i] = s.list[i];
  } else if (w.top_p < 1.0) {
    mass_bins<DT>(s, r, part.c0, part.c1);
    for (int i = t; i < kBins; i += kThreads) p.mass[(long long)blockIdx.x * kBins + i] = s.mass[i];
  }
}

// Without top-k: the stretches' masses, and the list.
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_cells_kernel(Sample p) {
  __shared__ Shared s;
  const int t = threadIdx.x;
  const long long b = blockIdx.x / p.S;
  const Want w(p, b);
  Row r = row_of<DT>(p, b);
  const Part part(p, r, b, blockIdx.x % p.S);
  const float largest = __uint_as_float((uint32_t)p.found[3 * b]);
  if (largest == -INFINITY || w.by_count) return;
  weigh(r, p, w, largest);
  if (needs_general(r, w)) return;
  int end = kBins;
  if (w.top_p < 1.0) {
    u64 m0 = 0, m1 = 0, base, total;
#pragma unroll
    for (int i = 0; i < kSplit; ++i)
      if (i < p.S) {
        m0 += p.mass[(b * p.S + i) * kBins + t];
        m1 += p.mass[(b * p.S + i) * kBins + t + kThreads];
      }
    s.mass[t] = m0;
    s.mass[t + kThreads] = m1;
    __syncthreads();
    end = end_bin(s, w.top_p, &base, &total);
    if (t == 0 && blockIdx.x % p.S == 0) {
      p.found[3 * b + 1] = base;
      p.found[3 * b + 2] = total;
    }
  }
  for (int c = part.c0 + t; c < part.c1; c += kThreads) s.cells[c] = 0;
  cell_sums<DT>(s, r, w, part.c0, part.c1, end);
  const uint32_t n = s.n;
  if (t == 0) p.counts[blockIdx.x] = n;
  for (uint32_t i = t; i < min(n, (uint32_t)kList); i += kThreads) p.list[(long long)blockIdx.x * kList + i] = s.list[i];
  for (int c = part.c0 + t; c < part.c1; c += kThreads) p.cells[b * kCells + c] = s.cells[c];
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(Sample p) {
  __shared__ Shared s;
  const int t = threadIdx.x;
  const long long b = blockIdx.x;
  // (All loads at once, wanted or not: each takes a microsecond.)
  uint32_t more[kSplit];
  u64 x[kSplit], cells[2];
#pragma unroll
  for (int i = 0; i < kSplit; ++i) {
    const long long part = b * p.S + min(i, p.S - 1);
    more[i] = p.counts[part];
    x[i] = p.list[part * kList + t];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) cells[i] = p.cells[b * kCells + t + i * kThreads];
  const u64 found[3] = {p.found[3 * b], p.found[3 * b + 1], p.found[3 * b + 2]};
  const Want w(p, b);
  Row r = row_of<DT>(p, b);
  const float largest = __uint_as_float((uint32_t)found[0]);
  if (none(p, b, largest)) return;
  weigh(r, p, w, largest);
  const bool limits = w.by_count || w.top_p < 1.0;
  bool plain = !needs_general(r, w);
  uint32_t n = 0;
  if (plain && limits) {
#pragma unroll
    for (int i = 0; i < kSplit; ++i) {
      if (i >= p.S) break;
      if ((uint32_t)t < more[i] && n + t < (uint32_t)kList) s.list[n + t] = x[i];
      for (uint32_t e = t + kThreads; e < more[i] && n + e < (uint32_t)kList; e += kThreads)
        s.list[n + e] = p.list[(b * p.S + i) * kList + e];
      n = min(n + more[i], (uint32_t)kList + 1);
    }
    plain = n <= (uint32_t)kList;
  }
  if (!plain) {
    hand_over<DT>(s, p, b, largest);
    return;
  }
  if (t == 0) s.n = n;
#pragma unroll
  for (int i = 0; i < 2; ++i) s.cells[t + i * kThreads] = !w.by_count && t + i * kThreads < r.cells ? cells[i] : 0;
  __syncthreads();
  const bool by_mass = limits && !w.by_count;
  finish<DT>(s, p, b, r, w, limits, by_mass ? found[1] : 0, by_mass ? found[2] : 0);
}

// Workgroups of a row: as many as give each CU one, up to kSplit, of 1024 pieces at least.
int split_of(int B, int V) {
  const long long pieces = V / kVec;
  return (int)std::max(1ll, std::min({(long long)kSplit, 256ll / B, pieces / kThreads}));
}

// Of the scratch memory: bytes of each part, and of all.
size_t lay_out(Sample* p, int B, char* at) {
  const size_t parts = (size_t)B * p->S;
  size_t used = 0;
  auto take = [&](size_t bytes) {
    char* const mine = at ? at + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return mine;
  };
  if (p->S == 1) return 0;
  p->maxima = reinterpret_cast<float*>(take(parts * kThreads * 4));
  p->mass = reinterpret_cast<u64*>(take(parts * kBins * 8));
  p->list = reinterpret_cast<u64*>(take(parts * kList * 8));
  p->cells = reinterpret_cast<u64*>(take((size_t)B * kCells * 8));
  p->counts = reinterpret_cast<uint32_t*>(take(parts * 4));
  p->found = reinterpret_cast<u64*>(take((size_t)B * 24));
  return used;
}

// Rows of a launch: a grid has less than 2^32 lanes.
constexpr int kRows = 1 << 21;

template <int DT>
void launch(const Sample& p, int B, hipStream_t st) {
  const dim3 block(kThreads);
  if (p.S == 1) {
    for (long long b = 0; b < B; b += kRows) {
      Sample q = p;
      q.x += b * p.xs;
      q.u = static_cast<const char*>(p.u) + b * (p.u64bits ? 8 : 4);
      q.out += b;
      if (q.logp) q.logp += b;
      if (q.temperatures) q.temperatures += b;
      if (q.top_ks) q.top_ks += b;
      if (q.top_ps) q.top_ps += b;
      if (q.min_ps) q.min_ps += b;
      hipLaunchKernelGGL(sample_kernel<DT>, dim3((unsigned)std::min<long long>(B - b, kRows)), block, 0, st, q);
    }
    return;
  }
  const dim3 grid((unsigned)(B * p.S));
  hipLaunchKernelGGL(sample_maxima_kernel<DT>, grid, block, 0, st, p);
  hipLaunchKernelGGL(sample_bins_kernel<DT>, grid, block, 0, st, p);
  hipLaunchKernelGGL(sample_cells_kernel<DT>, grid, block, 0, st, p);
  hipLaunchKernelGGL(sample_draw_kernel<DT>, dim3((unsigned)B), block, 0, st, p);
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" int dsqg_sample_workspace_size(int32_t B, int32_t V, int32_t dtype, size_t* bytes) {
  if (!bytes || B < 0 || V < 1 || (dtype != DSQG_F32 && dtype != DSQG_BF16 && dtype != DSQG_F16)) return DSQG_EINVAL;
  Sample p = {};
  p.S = B > 0 ? split_of(B, V) : 1;
  *bytes = lay_out(&p, B, nullptr);
  return DSQG_OK;
}

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
  p.bits = bits;
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
  p.S = split_of(a->B, a->V);
  if (lay_out(&p, a->B, static_cast<char*>(a->workspace)) > (a->workspace ? a->workspace_bytes : 0)) return DSQG_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return DSQG_EINVAL;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a->dtype == DSQG_F32) launch<DSQG_F32>(p, a->B, st);
  else if (a->dtype == DSQG_BF16) launch<DSQG_BF16>(p, a->B, st);
  else launch<DSQG_F16>(p, a->B, st);
  return hipGetLastError() == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
