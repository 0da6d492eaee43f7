// The paged cache's decode step on the matrix instructions (gfx950), for query heads that share a
// key/value head: up to sixteen of them are the columns of
//
//   S^T [rows x heads] = K Q^T,     O^T [D x heads] += V^T P^T
//
// in tiles of 32 rows, so that a key or value is read once for all of them and costs no vector
// instruction per head (dsqg_paged_decode.hip: one multiply-add each).
//
// A wave has a tile to itself.  Keys go from memory to the A operand as they are: lane (i, g) loads row i's
// elements at a step's k = 8 g (the order of the head dim inside the contraction is free, so 8-bit rows
// come in 16-byte pieces that serve two steps).  Values pass through the wave's LDS block, row-major, and
// come back transposed (ds_read_tr16_b64).  S^T's result layout (lane (j, g): head j, rows 4 g + r of both
// halves) is the B operand of the second product.  8-bit codes become bf16, which holds them exactly; the
// rows' scales multiply scores and weights in fp32.
//
// Roundings: the weights enter the second product as two 16-bit terms, w = hi + lo + O(2^-16 w) in bf16 and
// 2^-21 w in float16, down to two of its subnormal steps (weights are taken times 2^14 there, so that this is 2^-37
// of the largest); float16 queries against 8-bit keys are two bf16 terms, which hold them exactly.  Scores,
// statistics and sums are fp32.
//
// What bounds it: the cache's bytes, each read once (0.1 to 1.4 % more are fetched).  One sequence of
// 131072 positions, 8 heads of 64 in bfloat16 (268 MB): 41.7 us, 6.4 TB/s, what a copy's reads reach here; 64 of
// up to 8192, 8 x 4 heads of 128 over e4m3 (680 MB): 116 to 125 us; 32 of up to 2048, 12 heads of 64 (127 MB): 27;
// 16 of up to 16001, 1 x 8 heads of 96 (62 MB): 16.  The same kernel without its products takes the same time.
// What the short ones lose is the launch (3 us), two memory round trips and the last workgroup's wait: 8 heads of
// 32 over 77 positions take 3.5 us.  5 x 3 x 5 heads of 80 in float16 over int8, up to 5001 positions, take 9.3:
// 5.7 up to 16 positions, 7.1 in bfloat16 over bfloat16, the rest the conversions and the queries' second term.
// Against the vector instructions (dsqg_paged_decode.hip), which need a multiply-add for each head and element:
// four heads over e4m3 400 -> 132 us, eight of 96 94 -> 20, and also one head of 64, 38 -> 30 (the same steps
// otherwise).  A tile of 32 rows a wave leaves registers for four waves a SIMD (three above 64 elements), each with
// a tile in flight; eight and sixteen waves a workgroup, chunks placed by XCD and keys through LDS in whole rows
// were no faster, or slower.
#include <type_traits>

#include "dsqg_launch.hpp"
#include "dsqg_paged_tile.hpp"

namespace dsqg {
namespace {

// A workgroup's part: a unit, its rows from t0 on (at most `rows` of them), how many parts the unit has, and the
// number of this one.
struct Part {
  int b, hk, g0, t0, rows, n;
  int unit, count, at;
};

template <int QT, int CT, int D, bool SHARES>
__device__ __forceinline__ void attend_part(const PagedDecode& p, Part part, bf16_t (&sV)[kWaves][kTile * Geo<D>::RV],
                                            float (&wm)[kWaves][kMfmaHeads], float (&wl)[kWaves][kMfmaHeads]) {
  using S = Steps<CT, D>;
  using V = ValueMap<CT, D>;
  constexpr bool F16 = CT == DSQG_F16;                       // operands in float16 (else bf16)
  constexpr bool QLO = QT == DSQG_F16 && narrow(CT);         // queries in two terms
  constexpr int ES = elem_size(CT), KS = S::count, DB = D / 16, RV = Geo<D>::RV;

  const int b = part.b, hk = part.hk, g0 = part.g0;
  // (Opaque, so that what follows from it is worked out for each part and not held in registers across them.)
  const int l = opaque(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = l & 15, g = l >> 4;
  const int heads = min(kMfmaHeads, p.G - g0);

  // The page numbers of the wave's next 32 tiles, one half each lane: no load stands between a tile and its
  // rows.  They need no position (entries behind the sequence's last page may be no pages: their rows are
  // masked, whatever is said of them), so with chunks they are on their way together with it.
  const long long pos = SHARES ? 0 : load_const(p.pos + b);
  const int* table = p.c.table + b * p.c.ts;
  const int last = (p.c.M << p.c.shift) - 1;
  auto page_of = [&](int t) { return last < 0 ? -1 : load_const(table + (min((unsigned)t, (unsigned)last) >> p.c.shift)); };
  const int first = part.t0 + wave * kTile;
  auto pages_from = [&](int t) { return page_of(t + (l >> 1) * (kWaves * kTile) + 16 * (l & 1)); };
  const int page0[2] = {page_of(first), page_of(first + 16)};  // (scalar loads, before any vector one)
  int pages = pages_from(first);
  Raw8<QT> qraw[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    raw_zero<QT>(qraw[s]);
    const int d = S::at(s, g);
    if (i < heads && d < D) qraw[s] = raw_load<QT>(p.q + b * p.qb + (hk * p.G + g0 + i) * p.qh + d * elem_size(QT));
  }

  const int n = SHARES ? part.n : rows_at(p, pos);
  const int count = SHARES ? part.count : chunks_of(p, n);
  if (!SHARES && (int)blockIdx.y >= count) return;
  if (part.t0 == 0 && p.joins && threadIdx.x == 0) p.joins[part.unit] = make_int2(part.at, count);
  const long long h0 = (long long)b * p.H + hk * p.G + g0;  // first query head, in [B, H]
  if (n <= 0) {  // no rows: zeros; a position outside the table: NaN
    for (int e = threadIdx.x; e < heads * D; e += kBlock)
      store_out<QT>(p.out, h0 * D + e, n == 0 ? 0.f : __uint_as_float(0x7fc00000u));
    return;
  }
  const int t1 = min(part.t0 + part.rows, stored_of(p, n));

  // The wave's tile: key operands' bytes, value rows' pieces, scale bytes of rows 4 g + r of each half.  Loads
  // go through a buffer resource for each half's sixteen rows, so that a lane has one offset for all keys and
  // one for all values, and nothing outside those rows can be touched.
  Raw8<CT> kr[2][KS];
  uint4 vr[V::passes][V::per_lane];
  uint32_t eks[2] = {}, evs[2] = {};
  bool bad[2];
  const int kn = (int)p.c.kn, vn = (int)p.c.vn;
  const int klane = i * kn + g * (narrow(CT) && S::pairs > 0 ? 16 : 8 * ES);
  const int krest = i * kn + 8 * ES * g;  // the steps behind the pairs
  const int vlane = (l / V::lanes & 15) * vn + l % V::lanes * 16;
  bf16_t* const sVw = sV[wave];
  const bf16_t* const vtr = sVw + (4 * g + (i >> 2)) * RV + 4 * (i & 3);
  const long long kh = hk * p.c.kh, vh = hk * p.c.vh, ksh = hk * p.c.ksh, vsh = hk * p.c.vsh;

  auto load_as = [&](int k, auto aux) {  // the wave's tile k; aux: the loads' cache policy
    constexpr int AUX = decltype(aux)::value;
    const int tile = first + k * (kWaves * kTile);
    if ((k & 31) == 0 && k > 0) pages = pages_from(tile);
    __amdgpu_buffer_rsrc_t rk[2], rv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int page = k == 0 ? page0[h] : __builtin_amdgcn_readlane(pages, 2 * (k & 31) + h);
      bad[h] = (unsigned)page >= (unsigned)p.c.P;
      const unsigned at = bad[h] ? 0u : (unsigned)page;
      const unsigned slot = (unsigned)(tile + 16 * h) & ((1u << p.c.shift) - 1u);
      auto rows = [&](char* base, long long page_stride, int row_stride, long long head) {
        return __builtin_amdgcn_make_buffer_rsrc(
            base + (unsigned long long)at * (unsigned)page_stride + slot * (unsigned)row_stride + head, (short)0,
            15 * row_stride + D * ES, 0x00020000);
      };
      rk[h] = rows(p.c.k, p.c.kp, kn, kh);
      rv[h] = rows(p.c.v, p.c.vp, vn, vh);
      if constexpr (narrow(CT)) {
        auto bytes = [&](unsigned char* base, long long page_stride, long long head) {
          return __builtin_amdgcn_raw_buffer_load_b32(
              __builtin_amdgcn_make_buffer_rsrc(base + (unsigned long long)at * (unsigned)page_stride + slot + head, (short)0, 16,
                                                0x00020000), 4 * g, 0, 0);
        };
        eks[h] = bytes(p.c.ks, p.c.ksp, ksh);
        evs[h] = bytes(p.c.vs, p.c.vsp, vsh);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int q = 0; q < S::pairs; ++q) {
        if constexpr (narrow(CT)) {
          const uint4 x = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk[h], klane + 64 * q, 0, AUX));
          kr[h][2 * q].a = make_uint2(x.x, x.y);
          kr[h][2 * q + 1].a = make_uint2(x.z, x.w);
        }
      }
#pragma unroll
      for (int s = 2 * S::pairs; s < KS; ++s) {
        // (The elements behind a row's end, in its last step at D = 80, belong to the next row or to nobody.)
        constexpr bool cut = D % 32 != 0;
        const bool out = cut && s == KS - 1 && g >= D % 32 / 8;
        const int off = krest + (S::at(s, 0) * ES);
        if constexpr (narrow(CT)) kr[h][s].a = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rk[h], off, 0, AUX));
        else kr[h][s].a = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk[h], off, 0, AUX));
        if (out) raw_zero<CT>(kr[h][s]);
      }
    }
#pragma unroll
    for (int u = 0; u < V::passes; ++u) {
#pragma unroll
      for (int w = 0; w < V::per_lane; ++w) {
        // (A piece behind the row's end is not used.)
        const __amdgpu_buffer_rsrc_t r = rv[u * V::rows / 16];
        const int off = vlane + 16 * V::lanes * w, row = u * V::rows % 16 * vn;
        uint4 x = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, row, AUX));
        if constexpr (V::rows > 16) {  // both halves in one pass
          const uint4 y = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rv[1], off, row, AUX));
          if (l / V::lanes >= 16) x = y;
        }
        vr[u][w] = x;
      }
    }
  };

  auto load = [&](int k) {
    if (p.stream) load_as(k, std::integral_constant<int, 2>{});  // (non-temporal)
    else load_as(k, std::integral_constant<int, 0>{});
  };

  // The tile's value rows below `live` to LDS as operand values, zeros in the others' place.
  auto stage = [&](int live) {
    if (live < kTile) {
#pragma unroll
      for (int u = 0; u < V::passes; ++u)
#pragma unroll
        for (int w = 0; w < V::per_lane; ++w)
          if (u * V::rows + l / V::lanes >= live) vr[u][w] = zero16();
    }
#pragma unroll
    for (int u = 0; u < V::passes; ++u) {
      const int row = u * V::rows + l / V::lanes;
#pragma unroll
      for (int w = 0; w < V::per_lane; ++w) {
        const int piece = l % V::lanes + V::lanes * w;
        const uint4 x = vr[u][w];
        if (piece < V::pieces) {
          if constexpr (narrow(CT)) {
            Raw8<CT> lo, hi;
            lo.a = make_uint2(x.x, x.y);
            hi.a = make_uint2(x.z, x.w);
            st16(sVw + row * RV + 16 * piece, operand<CT>(lo));
            st16(sVw + row * RV + 16 * piece + 8, operand<CT>(hi));
          } else {
            st16(sVw + row * RV + 8 * piece, x);
          }
        }
      }
    }
  };


  if (first < t1) load(0);
  __builtin_amdgcn_sched_barrier(0);

  uint4 qh[KS], ql[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    if constexpr (QLO) {
      float x[8];
      raw_floats<QT>(qraw[s], x);
      split8(x, qh[s], ql[s]);
    } else {
      qh[s] = qraw[s].a;
    }
  }

  // Scores of 16 rows (A operands in a), before any scale.
  auto scores = [&](const Raw8<CT> (&a)[KS]) {
    f32x4_t s = zero4();
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const uint4 x = operand<CT>(a[k]);
      s = mfma32<F16>(x, qh[k], s);
      if constexpr (QLO) s = mfma32<F16>(x, ql[k], s);
    }
    return s;
  };

  float m, lsum;  // of head i: the weights' reference exponent, the sum over this lane's rows
  f32x4_t o[DB];
  const float nan = __uint_as_float(0x7fc00000u);

  m = -INFINITY;
  lsum = 0.f;
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = zero4();

  if (p.kn && part.t0 == 0 && wave == kWaves - 1) {
    // The new row is the first part's last wave's (no other has fewer tiles, and later parts would end later for
    // it: 32 sequences of up to 2048, 30.5 -> 32.3 us).  It begins the statistics: its score is row 0 of a product
    // whose other rows are zeros, its weight is the reference's.
    const int t = n - 1, at = __builtin_amdgcn_readfirstlane(page_of(t));
    const bool ok = (unsigned)at < (unsigned)p.c.P, keep = ok && i == 0 && g0 == 0;
    const long long slot = t & ((1 << p.c.shift) - 1);
    const char* src = p.kn + b * p.knb + hk * p.knh;
    char* dst = p.c.k + at * p.c.kp + kh + slot * p.c.kn;
    // (Kept out of registers during the tiles.)
    asm volatile("" : "+s"(src), "+s"(dst));
    float x;
    {
      Raw8<CT> kc[KS];
      int byte = 127;
      Raw8<QT> r[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        raw_zero<QT>(r[s]);
        if (S::at(s, g) < D) r[s] = raw_load<QT>(src + S::at(s, g) * elem_size(QT));
      }
      if constexpr (narrow(CT)) {
        float f[8], mk = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          raw_floats<QT>(r[s], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) mk = max_nan(mk, fabsf(f[e]));
        }
        mk = max_nan(mk, __shfl_xor(mk, 16, 64));
        byte = scale_byte<CT>(max_nan(mk, __shfl_xor(mk, 32, 64)));
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          raw_floats<QT>(r[s], f);
          kc[s] = raw_encode<CT>(f, byte);
        }
        if (keep && g == 0) p.c.ks[at * p.c.ksp + ksh + slot] = (unsigned char)byte;
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) kc[s].a = r[s].a;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if (keep && S::at(s, g) < D) raw_store<CT>(dst + S::at(s, g) * ES, kc[s]);
        if (i != 0) raw_zero<CT>(kc[s]);
      }
      x = scores(kc)[0];
      if constexpr (narrow(CT)) x *= scale_value(byte);
    }
    x = __shfl(x, i, 64) * p.scale;  // (row 0 is in the lanes of g = 0)
    if (!ok) x = nan;
    m = lifted<F16>(fmaxf(x, -INFINITY));
    const float e = weight(x, m);
    lsum = g == 0 ? e : 0.f;
    // Values in the result's layout: four elements at 16 d + 4 g.
    src = p.vn + b * p.vnb + hk * p.vnh;
    dst = p.c.v + at * p.c.vp + vh + slot * p.c.vn;
    asm volatile("" : "+s"(src), "+s"(dst));
    uint2 y[DB];
    float mv = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      y[d] = *reinterpret_cast<const uint2*>(src + (16 * d + 4 * g) * elem_size(QT));
      Raw8<QT> r;
      float f[8];
      r.a = make_uint4(y[d].x, y[d].y, 0u, 0u);
      raw_floats<QT>(r, f);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mv = max_nan(mv, fabsf(f[q]));
        o[d][q] = f[q];
      }
    }
    if constexpr (narrow(CT)) {
      mv = max_nan(mv, __shfl_xor(mv, 16, 64));
      const int byte = scale_byte<CT>(max_nan(mv, __shfl_xor(mv, 32, 64)));
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        float f[8] = {o[d][0], o[d][1], o[d][2], o[d][3], 0.f, 0.f, 0.f, 0.f};
        const Raw8<CT> c = raw_encode<CT>(f, byte);
        if (keep) *reinterpret_cast<uint32_t*>(dst + 16 * d + 4 * g) = c.a.x;
        raw_floats<CT>(c, f);
#pragma unroll
        for (int q = 0; q < 4; ++q) o[d][q] = f[q] * scale_value(byte);
      }
      if (keep && g == 0) p.c.vs[at * p.c.vsp + vsh + slot] = (unsigned char)byte;
    } else if (keep) {
#pragma unroll
      for (int d = 0; d < DB; ++d) *reinterpret_cast<uint2*>(dst + (16 * d + 4 * g) * ES) = y[d];
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] *= e;
  }

#pragma unroll 1
  for (int k = 0, tile = first; tile < t1; ++k, tile += kWaves * kTile) {
    const int live = t1 - tile;
    const f32x4_t s0 = scores(kr[0]), s1 = scores(kr[1]);
    __builtin_amdgcn_wave_barrier();
    stage(live);
    const uint32_t ek[2] = {eks[0], eks[1]}, ev[2] = {evs[0], evs[1]};
    const bool no[2] = {bad[0], bad[1]};
    // The next tile's rows are on their way during the softmax and the second product.
    if (tile + kWaves * kTile < t1) load(k + 1);
    __builtin_amdgcn_sched_barrier(0);

    float x[8], w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = (e < 4 ? s0[e % 4] : s1[e % 4]) * p.scale;
      if constexpr (narrow(CT)) x[e] = __builtin_amdgcn_ldexpf(x[e], (int)((ek[e / 4] >> (8 * (e % 4))) & 255) - 127);
    }
    // (255 - byte is zero nowhere, by the usual test of a word's bytes, unless a row reads as NaN.)
    bool odd = false;
    if constexpr (narrow(CT))
      odd = __any((((0xfefefefeu - ek[0]) & ek[0]) | ((0xfefefefeu - ek[1]) & ek[1]) | ((0xfefefefeu - ev[0]) & ev[0]) |
                   ((0xfefefefeu - ev[1]) & ev[1])) & 0x80808080u);
    if (odd | no[0] | no[1]) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (no[e / 4] || (narrow(CT) && ((ek[e / 4] >> (8 * (e % 4))) & 255) == 255)) x[e] = nan;
    }
    if (live < kTile) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 16 * (e / 4) + 4 * g + e % 4 < live ? x[e] : -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
    mx = lifted<F16>(col_max(mx));
    if (__any(mx > m)) {
      const float mn = fmaxf(m, mx), a = weight(m, mn);
      m = mn;
      lsum *= a;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= a;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = weight(x[e], m);
    if (live < kTile) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 16 * (e / 4) + 4 * g + e % 4 < live ? w[e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) lsum += w[e];
    if constexpr (narrow(CT)) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __builtin_amdgcn_ldexpf(w[e], (int)((ev[e / 4] >> (8 * (e % 4))) & 255) - 127);
      if (odd) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (((ev[e / 4] >> (8 * (e % 4))) & 255) == 255) f[e] = nan;
      }
      if (live < kTile) {  // (a scale behind the last row is no number of this sequence)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 16 * (e / 4) + 4 * g + e % 4 < live ? f[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = f[e];
    }
    uint4 hi, lo;
    split_weights<F16, !narrow(CT)>(w, hi, lo);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the rows are staged
    __builtin_amdgcn_wave_barrier();
    auto values = [&](int d) {
      const uint2 a = __builtin_bit_cast(uint2, lds_read_tr16(vtr + 16 * d));
      const uint2 c = __builtin_bit_cast(uint2, lds_read_tr16(vtr + 16 * RV + 16 * d));
      return make_uint4(a.x, a.y, c.x, c.y);
    };
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const uint4 v = values(d);
      o[d] = mfma32<F16>(v, hi, o[d]);
      o[d] = mfma32<F16>(v, lo, o[d]);
      if (d % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }

  // The waves' parts meet in LDS, each in its own block.
  lsum = col_sum(lsum);
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_wave_barrier();
  float* const sums = reinterpret_cast<float*>(sVw);  // [16][D]
  static_assert(kMfmaHeads * D * 4 <= kTile * RV * 2, "a wave's part fits its block");
#pragma unroll
  for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4_t*>(sums + i * D + 16 * d + 4 * g) = o[d];
  if (g == 0) {
    wm[wave][i] = m;
    wl[wave][i] = lsum;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < heads * D; e += kBlock) {
    const int h = e / D, d = e - h * D;
    float mm = -INFINITY, ll = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, wm[w][h]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float a = weight(wm[w][h], mm);
      ll = fmaf(wl[w][h], a, ll);
      x = fmaf(reinterpret_cast<const float*>(sV[w])[e], a, x);
    }
    if (count == 1) {
      store_out<QT>(p.out, h0 * D + e, x / ll);
    } else {
      const long long at = (long long)part.at * p.heads + h;
      p.acc[at * D + d] = x;
      if (d == 0) {
        p.ml[2 * at] = mm;
        p.ml[2 * at + 1] = ll;
      }
    }
  }
}

// Workgroups that a CU holds: by registers four waves a SIMD where rows are short, else three.
constexpr int places(int D) { return D <= 64 ? 4 : 3; }

template <int QT, int CT, int D, bool SHARES>
__global__ __launch_bounds__(kBlock, places(D)) void paged_mfma_kernel(PagedDecode p) {
  __shared__ __align__(16) bf16_t sV[kWaves][kTile * Geo<D>::RV];
  __shared__ float wm[kWaves][kMfmaHeads], wl[kWaves][kMfmaHeads];
  const int ht = (p.G + kMfmaHeads - 1) / kMfmaHeads;
  const int units = p.c.Hkv * ht;
  auto unit = [&](Part& part, int u) {  // unit u of sequence part.b
    part.unit = part.b * units + u;
    part.hk = u / ht;
    part.g0 = (u - part.hk * ht) * kMfmaHeads;
  };
  Part part;
  if constexpr (!SHARES) {
    part.b = blockIdx.x / units;
    unit(part, blockIdx.x - part.b * units);
    part.t0 = blockIdx.y * p.chunk;
    part.rows = p.chunk;
    part.at = blockIdx.x * p.splits + blockIdx.y;
    attend_part<QT, CT, D, false>(p, part, sV, wm, wl);
  } else {
    const int w = blockIdx.x;
    int s, end, begin, per;
    {
      const ShareLine line(p);
      per = line.per;
      s = w * per;
      end = min(s + per, line.steps());
      if (s >= end) return;
      part.b = line.sequence(p, s);
      part.n = line.rows(part.b);
      begin = line.before(p, part.b);
    }
#pragma unroll 1
    while (true) {
      const int steps = steps_of(p, part.n), u = (s - begin) / steps, at = s - begin - u * steps;
      const int take = min(end - s, steps - at);
      unit(part, u);
      part.t0 = at * kShareRows;
      part.rows = take * kShareRows;
      part.at = w + part.unit;
      // (Of the unit's first part, the count; of the others, whether they are all.)
      part.count = at == 0 ? (s + steps - 1) / per - w + 1 : 2;
      attend_part<QT, CT, D, true>(p, part, sV, wm, wl);
      s += take;
      if (s >= end) break;
      if (s == begin + steps * units) {
        part.n = rows_of(p, ++part.b);
        begin = s;
      }
      __syncthreads();  // (the next part's values go where this one's sums were read)
    }
  }
}

template <int QT, int CT, int D>
void launch(const PagedDecode& p, hipStream_t st) {
  if constexpr (paged_mfma_shares(CT, D)) {
    if (p.shares) {
      hipLaunchKernelGGL((paged_mfma_kernel<QT, CT, D, true>), dim3((unsigned)p.shares), dim3(kBlock), 0, st, p);
      return;
    }
  }
  const unsigned units = (unsigned)(p.c.B * p.c.Hkv * ((p.G + kMfmaHeads - 1) / kMfmaHeads));
  hipLaunchKernelGGL((paged_mfma_kernel<QT, CT, D, false>), dim3(units, (unsigned)p.splits), dim3(kBlock), 0, st, p);
}

template <int QT, int CT>
void launch_dim(const PagedDecode& p, int D, hipStream_t st) {
  switch (D) {
    case 32: launch<QT, CT, 32>(p, st); break;
    case 64: launch<QT, CT, 64>(p, st); break;
    case 80: launch<QT, CT, 80>(p, st); break;
    case 96: launch<QT, CT, 96>(p, st); break;
    default: launch<QT, CT, 128>(p, st); break;
  }
}

}  // namespace

bool paged_mfma_takes(const PagedDecode& p, int dtype, int cache_dtype) {
  if (dtype == DSQG_F32) return false;
  if (!narrow(cache_dtype)) return true;
  // Scale bytes come four at a time, at 32-bit offsets from page to page.
  const long long odd = p.c.ksp | p.c.ksh | p.c.vsp | p.c.vsh | (long long)reinterpret_cast<uintptr_t>(p.c.ks) |
                        (long long)reinterpret_cast<uintptr_t>(p.c.vs);
  return p.c.ksn == 1 && p.c.vsn == 1 && odd % 4 == 0 && p.c.ksp < (1ll << 31) && p.c.vsp < (1ll << 31);
}

int paged_mfma_places(int D) { return 256 * places(D); }

void launch_paged_mfma(const PagedDecode& p, int dtype, int cache_dtype, int D, hipStream_t st) {
  if (dtype == DSQG_BF16) {
    if (cache_dtype == DSQG_E4M3) launch_dim<DSQG_BF16, DSQG_E4M3>(p, D, st);
    else if (cache_dtype == DSQG_INT8) launch_dim<DSQG_BF16, DSQG_INT8>(p, D, st);
    else launch_dim<DSQG_BF16, DSQG_BF16>(p, D, st);
  } else {
    if (cache_dtype == DSQG_E4M3) launch_dim<DSQG_F16, DSQG_E4M3>(p, D, st);
    else if (cache_dtype == DSQG_INT8) launch_dim<DSQG_F16, DSQG_INT8>(p, D, st);
    else launch_dim<DSQG_F16, DSQG_F16>(p, D, st);
  }
}

}  // namespace dsqg
