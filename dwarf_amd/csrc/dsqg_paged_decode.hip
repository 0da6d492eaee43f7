// Attention of one new token per sequence over a paged key/value cache (gfx950): the plan, the kernel of the
// vector instructions and the join.
//
//   out[h] = sum_t w_t v_t,  w = softmax_t(scale q_h . k_t),  t = 0 .. pos
//
// One pass over the rows with a running maximum and sum: of the rows seen so far a group of lanes keeps
// m = max s_t, l = sum 2^(s_t - m) and acc = sum 2^(s_t - m) v_t (scores in base 2), and the parts of
// different rows join as  acc = sum_i 2^(m_i - m) acc_i.  (m carries an offset, weight_lift: the largest weight
// is not 1.)  Every key and value is read once for each group of up to 1, 2 or 4 query heads that share it
// (plan's p.heads), so memory bounds the step, and short ones the launches and the round trips from the position to
// the rows; the groups of one key/value head are neighbouring workgroups, which lie on different XCDs.
//
// 16-bit queries take the matrix instructions (dsqg_paged_mfma.hip, with the figures of long steps).  The kernel
// here takes float32 ones, whose products the 16-bit instructions would round (those of float32 operands would
// not, but have sixteen columns for what is one head in the float32 steps that are listed; with many heads they
// would read the pages once where this kernel reads them for each group: not built), and 8-bit pools whose scales
// the other kernel cannot read four at a time.  4 float32 sequences of up to 2048 positions, 8 heads of 32 (10 MB):
// 5.2 us and 3.7 for the join; a launch alone is about 3 of each.
//
// Its workgroup has one key/value head of one sequence, up to GT of the query heads that share it, and a
// chunk of the sequence's rows; its four waves take tiles in turn.  In a tile a row is 4, 8 or 16
// neighbouring lanes (RowMap), each wave load being whole rows of one page: a tile starts at a multiple of
// the wave's rows and a page is a multiple of them too.  Row groups keep statistics of their own until the
// chunk's end.  The first chunk's workgroup takes the new row from the caller's k_new and v_new (as the cache
// will hold it: through the 8-bit type's rounding), and stores it; no workgroup reads that row from the pool.
#include <algorithm>

#include "dsqg_launch.hpp"
#include "dsqg_mfma.hpp"
#include "dsqg_paged.hpp"

namespace dsqg {
namespace {

constexpr int kWaves = kBlock / 64;

// a + sum of the products of eight queries and eight key elements.
template <int CT>
__device__ __forceinline__ float dot8(const float (&q)[8], const Raw8<CT>& kr, float a) {
  float k[8];
  raw_floats<CT>(kr, k);
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaf(q[i], k[i], a);
  return a;
}

// Statistics and output sums of GT heads over the rows of one lane group.
template <int GT, int PC>
struct Running {
  float m[GT], l[GT], acc[GT][PC][8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int u = 0; u < PC; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[g][u][i] = 0.f;
    }
  }
};

template <int QT, int CT, int D, int GT>
__global__ __launch_bounds__(kBlock) void paged_decode_kernel(PagedDecode p) {
  using R = RowMap<D>;
  constexpr int PC = R::pieces, ES = elem_size(CT);
  constexpr int U = CT == DSQG_F32 || PC > 1 ? 2 : 4;  // passes of a tile
  constexpr int TR = U * R::rows, stride = kWaves * TR;
  const int hg = (p.G + GT - 1) / GT;
  const int b = blockIdx.x / (p.c.Hkv * hg), rest = blockIdx.x - b * p.c.Hkv * hg;
  const int hk = rest / hg, g0 = (rest - hk * hg) * GT;
  const int split = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int gl = lane % R::lanes, r = lane / R::lanes;

  // The page numbers of the wave's next 64 / U tiles, a pass each lane: no load stands between a tile and its
  // rows.  Like the queries they need no position (entries behind the sequence's last page may be no pages:
  // their rows are masked, whatever is said of them), so all of them are on their way together.
  const int* table = p.c.table + b * p.c.ts;
  const int last = (p.c.M << p.c.shift) - 1;
  auto page_of = [&](int t) { return last < 0 ? -1 : load_const(table + (min((unsigned)t, (unsigned)last) >> p.c.shift)); };
  const int t0 = split * p.chunk, first = t0 + wave * TR;
  auto pages_from = [&](int t) { return page_of(t + lane / U * stride + lane % U * R::rows); };
  int pages = pages_from(first);

  float q[GT][PC][8];
#pragma unroll
  for (int g = 0; g < GT; ++g)
#pragma unroll
    for (int u = 0; u < PC; ++u) {
      const int piece = gl + R::lanes * u;
      Raw8<QT> x;
      raw_zero<QT>(x);
      if (g0 + g < p.G && piece < R::CPR)
        x = raw_load<QT>(p.q + b * p.qb + (hk * p.G + g0 + g) * p.qh + piece * 8 * elem_size(QT));
      raw_floats<QT>(x, q[g][u]);
    }

  const int n = rows_of(p, b);
  const int chunks = chunks_of(p, n);
  if (split >= chunks) return;
  if (split == 0 && p.joins && threadIdx.x == 0) p.joins[blockIdx.x] = make_int2(blockIdx.x * p.splits, chunks);
  const long long h0 = (long long)b * p.H + hk * p.G + g0;  // first query head, in [B, H]
  if (n <= 0) {  // no rows: zeros; a position outside the table: NaN
    for (int e = threadIdx.x; e < GT * D; e += kBlock)
      if (g0 + e / D < p.G) store_out<QT>(p.out, h0 * D + e, n == 0 ? 0.f : __uint_as_float(0x7fc00000u));
    return;
  }
  const bool fresh = p.kn != nullptr;
  const int t1 = min(t0 + p.chunk, stored_of(p, n));

  // The wave's tile k.  Loads go through a buffer resource for each pass's rows, so that nothing outside them
  // can be touched.  (A pass that lies behind the last row is masked.)
  Raw8<CT> kr[U][PC], vr[U][PC];
  int sk[U], sv[U];  // scale bytes
  bool bad[U];
  auto place = [&](int k, int u, unsigned& at, unsigned& slot) {
    const int t = first + k * stride + u * R::rows, page = __builtin_amdgcn_readlane(pages, k % (64 / U) * U + u);
    bad[u] = (unsigned)page >= (unsigned)p.c.P;
    at = bad[u] ? 0u : (unsigned)page;
    slot = (unsigned)t & ((1u << p.c.shift) - 1u);
  };
  auto load_rows = [&](Raw8<CT> (&x)[PC], const char* base, int row) {
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, (R::rows - 1) * row + D * ES, 0x00020000);
#pragma unroll
    for (int w = 0; w < PC; ++w) {
      // (A piece behind the row's end, at D = 80, is another row's or nobody's.)
      const int off = r * row + (gl + R::lanes * w) * 8 * ES;
      if constexpr (narrow(CT)) {
        x[w].a = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, 0, 0));
      } else {
        x[w].a = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0));
        if constexpr (CT == DSQG_F32) x[w].b = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + 16, 0, 0));
      }
      if (gl + R::lanes * w >= R::CPR) raw_zero<CT>(x[w]);
    }
  };
  auto load_k = [&](int k) {
    if (k > 0 && k % (64 / U) == 0) pages = pages_from(first + k * stride);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unsigned at, slot;
      place(k, u, at, slot);
      load_rows(kr[u], p.c.k + at * p.c.kp + hk * p.c.kh + slot * p.c.kn, (int)p.c.kn);
      if constexpr (narrow(CT)) sk[u] = p.c.ks[at * p.c.ksp + hk * p.c.ksh + (slot + r) * p.c.ksn];
    }
  };
  auto load_v = [&](int k) {  // (after load_k of the same tile)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unsigned at, slot;
      place(k, u, at, slot);
      load_rows(vr[u], p.c.v + at * p.c.vp + hk * p.c.vh + slot * p.c.vn, (int)p.c.vn);
      if constexpr (narrow(CT)) sv[u] = p.c.vs[at * p.c.vsp + hk * p.c.vsh + (slot + r) * p.c.vsn];
    }
  };
  if (first < t1) {
    load_k(0);
    load_v(0);
  }

  Running<GT, PC> s;
  s.clear();

  // The new row, in the first row group of the first chunk's last wave (no other has fewer tiles).
  if (fresh && split == 0 && wave == kWaves - 1) {
    const char* kn = p.kn + b * p.knb + hk * p.knh;
    const char* vn = p.vn + b * p.vnb + hk * p.vnh;
    Raw8<QT> x[PC], y[PC];
#pragma unroll
    for (int u = 0; u < PC; ++u) {
      const int piece = gl + R::lanes * u;
      raw_zero<QT>(x[u]);
      raw_zero<QT>(y[u]);
      if (piece < R::CPR) {
        x[u] = raw_load<QT>(kn + piece * 8 * elem_size(QT));
        y[u] = raw_load<QT>(vn + piece * 8 * elem_size(QT));
      }
    }
    Raw8<CT> kc[PC], vc[PC];
    int kb = 0, vb = 0;
    if constexpr (narrow(CT)) {
      float f[PC][8], w[PC][8], mk = 0.f, mv = 0.f;
#pragma unroll
      for (int u = 0; u < PC; ++u) {
        raw_floats<QT>(x[u], f[u]);
        raw_floats<QT>(y[u], w[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          mk = max_nan(mk, fabsf(f[u][i]));
          mv = max_nan(mv, fabsf(w[u][i]));
        }
      }
      kb = scale_byte<CT>(group_max_nan<R::lanes>(mk));
      vb = scale_byte<CT>(group_max_nan<R::lanes>(mv));
#pragma unroll
      for (int u = 0; u < PC; ++u) {
        kc[u] = raw_encode<CT>(f[u], kb);
        vc[u] = raw_encode<CT>(w[u], vb);
      }
    } else {
#pragma unroll
      for (int u = 0; u < PC; ++u) {
        kc[u] = x[u];
        vc[u] = y[u];
      }
    }
    const int t = n - 1, page = page_of(t);
    const bool ok = (unsigned)page < (unsigned)p.c.P;
    const float sk = narrow(CT) ? scale_value(kb) : 1.f, sv = narrow(CT) ? scale_value(vb) : 1.f;
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float d = 0.f;
#pragma unroll
      for (int u = 0; u < PC; ++u) d = dot8<CT>(q[g][u], kc[u], d);
      d = group_sum<R::lanes>(d) * (p.scale * sk);
      if (!ok) d = __uint_as_float(0x7fc00000u);  // nowhere to keep the row
      if (r == 0) {
        s.m[g] = lifted<false>(fmaxf(d, -INFINITY));
        s.l[g] = weight(d, s.m[g]);
#pragma unroll
        for (int u = 0; u < PC; ++u) {
          float v[8];
          raw_floats<CT>(vc[u], v);
#pragma unroll
          for (int i = 0; i < 8; ++i) s.acc[g][u][i] = s.l[g] * sv * v[i];
        }
      }
    }
    if (ok && r == 0 && g0 == 0) {
      const long long slot = t & ((1 << p.c.shift) - 1);
      char* kd = p.c.k + page * p.c.kp + hk * p.c.kh + slot * p.c.kn;
      char* vd = p.c.v + page * p.c.vp + hk * p.c.vh + slot * p.c.vn;
#pragma unroll
      for (int u = 0; u < PC; ++u) {
        const int piece = gl + R::lanes * u;
        if (piece < R::CPR) {
          raw_store<CT>(kd + piece * 8 * ES, kc[u]);
          raw_store<CT>(vd + piece * 8 * ES, vc[u]);
        }
      }
      if constexpr (narrow(CT)) {
        if (gl == 0) {
          p.c.ks[page * p.c.ksp + hk * p.c.ksh + slot * p.c.ksn] = (unsigned char)kb;
          p.c.vs[page * p.c.vsp + hk * p.c.vsh + slot * p.c.vsn] = (unsigned char)vb;
        }
      }
    }
  }

#pragma unroll 1
  for (int k = 0, tile = first; tile < t1; ++k, tile += stride) {
    const bool more = tile + stride < t1;
    float sc[GT][U];
    bool no[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      no[u] = bad[u];
      const float c = narrow(CT) ? p.scale * scale_value(sk[u]) : p.scale;
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        float d = 0.f;
#pragma unroll
        for (int w = 0; w < PC; ++w) d = dot8<CT>(q[g][w], kr[u][w], d);
        sc[g][u] = group_sum<R::lanes>(d) * c;
        if (no[u]) sc[g][u] = __uint_as_float(0x7fc00000u);
      }
    }
    // The next tile's keys are on their way during the softmax, its values during the next scores.
    if (more) load_k(k + 1);
    if (tile + TR > t1) {
      // What lies behind the last row is no number of this sequence: zeros, so that 0 * value is 0.
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (tile + u * R::rows + r >= t1) {
          sv[u] = 127;
#pragma unroll
          for (int g = 0; g < GT; ++g) sc[g][u] = -INFINITY;
#pragma unroll
          for (int w = 0; w < PC; ++w) raw_zero<CT>(vr[u][w]);
        }
    }
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float m = sc[g][0];
#pragma unroll
      for (int u = 1; u < U; ++u) m = fmaxf(m, sc[g][u]);
      m = fmaxf(s.m[g], lifted<false>(m));
      const float a = weight(s.m[g], m);
      s.m[g] = m;
      s.l[g] *= a;
#pragma unroll
      for (int w = 0; w < PC; ++w)
#pragma unroll
        for (int i = 0; i < 8; ++i) s.acc[g][w][i] *= a;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = weight(sc[g][u], m);
        s.l[g] += e;
        sc[g][u] = narrow(CT) ? e * scale_value(sv[u]) : e;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int w = 0; w < PC; ++w) {
        float x[8];
        raw_floats<CT>(vr[u][w], x);
#pragma unroll
        for (int g = 0; g < GT; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) s.acc[g][w][i] = fmaf(sc[g][u], x[i], s.acc[g][w][i]);
      }
    if (more) load_v(k + 1);
  }

  // The row groups of the wave, then the waves through LDS.
  __shared__ float wm[kWaves][GT], wl[kWaves][GT], wacc[kWaves][GT][D];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    float m = s.m[g];
#pragma unroll
    for (int x = R::lanes; x < 16; x *= 2) m = fmaxf(m, __shfl_xor(m, x, 64));
    m = col_max(m);
    const float a = weight(s.m[g], m);
    float l = s.l[g] * a;
#pragma unroll
    for (int x = R::lanes; x < 16; x *= 2) l += __shfl_xor(l, x, 64);
    l = col_sum(l);
    if (lane == 0) {
      wm[wave][g] = m;
      wl[wave][g] = l;
    }
#pragma unroll
    for (int w = 0; w < PC; ++w)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x = s.acc[g][w][i] * a;
#pragma unroll
        for (int y = R::lanes; y < 16; y *= 2) x += __shfl_xor(x, y, 64);
        x = col_sum(x);
        const int piece = gl + R::lanes * w;
        if (r == 0 && piece < R::CPR) wacc[wave][g][piece * 8 + i] = x;
      }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < GT * D; e += kBlock) {
    const int g = e / D, d = e - g * D;
    if (g0 + g >= p.G) break;
    float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, wm[w][g]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float a = weight(wm[w][g], m);
      l = fmaf(wl[w][g], a, l);
      x = fmaf(wacc[w][g][d], a, x);
    }
    if (chunks == 1) {
      store_out<QT>(p.out, h0 * D + e, x / l);
    } else {
      const long long at = ((long long)blockIdx.x * p.splits + split) * p.heads + g;
      p.acc[at * D + d] = x;
      if (d == 0) {
        p.ml[2 * at] = m;
        p.ml[2 * at + 1] = l;
      }
    }
  }
}

// Joins a head's parts.  Grid: [units * heads].  A part is JL lanes of four elements; the workgroup's rows of
// lanes take parts in turn, each with a running maximum of its own, and meet in LDS: the order is fixed by the
// sequences' lengths.  Of chunks it is known beforehand where they are, so that one memory round trip brings how
// many there are and the first of them; of shares, two.
template <int QT, int D>
__global__ __launch_bounds__(1024) void paged_join_kernel(PagedDecode p) {
  constexpr int JL = D <= 32 ? 8 : D <= 64 ? 16 : 32, U = 4;
  const int unit = blockIdx.x / p.heads, h = blockIdx.x - unit * p.heads, rows = blockDim.x / JL;
  const int gl = threadIdx.x % JL, r = threadIdx.x / JL;
  const int units = (p.G + p.heads - 1) / p.heads;  // of a key/value head
  const int bk = unit / units, hq = (unit - bk * units) * p.heads + h;
  if (hq >= p.G) return;
  const long long head = (long long)bk * p.G + hq;
  float2 s[U];
  float4 v[U];
  const float2* ml = reinterpret_cast<const float2*>(p.ml) + h;
  const float* acc = p.acc + (long long)h * D + 4 * gl;
  auto load = [&](long long first, int c0, int parts) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * rows;
      s[u] = make_float2(-INFINITY, 0.f);
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < parts) {
        s[u] = ml[(first + c) * p.heads];
        if (4 * gl < D) v[u] = *reinterpret_cast<const float4*>(acc + (first + c) * p.heads * D);
      }
    }
  };
  const bool chunked = p.shares == 0;
  if (chunked) load((long long)unit * p.splits, r, p.splits);
  const int2 join = p.joins[unit];
  const int parts = join.y;
  if (parts == 1) return;  // (written by its only workgroup)
  if (!chunked) load(join.x, r, parts);
  float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = r;;) {
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + u * rows >= parts) {  // (what lies behind the last part was never written)
        s[u] = make_float2(-INFINITY, 0.f);
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      mn = fmaxf(mn, s[u].x);
    }
    const float a = weight(m, mn);
    m = mn;
    l *= a;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= a;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = weight(s[u].x, m);
      l = fmaf(s[u].y, w, l);
      x[0] = fmaf(v[u].x, w, x[0]);
      x[1] = fmaf(v[u].y, w, x[1]);
      x[2] = fmaf(v[u].z, w, x[2]);
      x[3] = fmaf(v[u].w, w, x[3]);
    }
    c0 += U * rows;
    if (c0 >= parts) break;
    load(join.x, c0, parts);
  }
  __shared__ float jm[1024 / JL], jl[1024 / JL], jx[1024 / JL][D];
  if (4 * gl < D)
#pragma unroll
    for (int i = 0; i < 4; ++i) jx[r][4 * gl + i] = x[i];
  if (gl == 0) {
    jm[r] = m;
    jl[r] = l;
  }
  __syncthreads();
  const int n = min(rows, parts);
  m = -INFINITY;
  for (int i = 0; i < n; ++i) m = fmaxf(m, jm[i]);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float o = 0.f;
    l = 0.f;
    for (int i = 0; i < n; ++i) {
      const float w = weight(jm[i], m);
      l = fmaf(jl[i], w, l);
      o = fmaf(jx[i][d], w, o);
    }
    store_out<QT>(p.out, head * D + d, o / l);
  }
}

long long units_of(const PagedDecode& p) { return (long long)p.c.B * p.c.Hkv * ((p.G + p.heads - 1) / p.heads); }

// Chooses the kernel (true: matrix instructions) and the split; returns the parts (of `heads` each) that may have
// to be joined.
long long plan(PagedDecode& p, int dtype, int cache_dtype, int D, bool* mfma) {
  *mfma = dtype != DSQG_F32 && paged_mfma_takes(p, dtype, cache_dtype);
  // Four heads of the vector kernel take 146 to 155 registers, three waves a SIMD; at D = 80 and 96, three groups
  // of eight a lane, two heads take 178 to 212 over 8 bits (two waves) and all 256 over float32 (one wave).
  p.heads = *mfma ? std::min(p.G, kMfmaHeads) : p.G == 1 ? 1 : p.G == 2 || D == 80 || D == 96 ? 2 : 4;
  const bool small = narrow(cache_dtype);
  const long long T = std::max(1ll, (long long)p.c.M << p.c.shift);
  const long long units = units_of(p), steps = units * ((T + kShareRows - 1) / kShareRows);
  // (The vector kernel's is a number of workgroups that chunks were found to be well cut for, six a CU; by registers
  // a CU holds five of one head, four of two and three of four, at D = 80 and 96 four to one.)
  const long long places = *mfma ? paged_mfma_places(D) : 1536;
  p.shares = p.splits = 0;
  // T is what the table holds, for the host knows no positions.  Under a table longer than its sequences the split is
  // the table's: 8 heads of 32 at 77 positions 3.6 us (in a replayed graph) under a table of 128 or 512, 5.5 under
  // 2048; 8 of 64 at 8000 10.4 under 8064, 13.1 under 131072; 16 x 8 x 4 of 128 at 4000 50.9 under 4032, 69.0 under
  // 32768.
  // One workgroup for each unit needs no second launch: it pays until a unit's rows take longer than that and, where
  // units fill the chip, longer.  In one / in parts, us, 1 unit: 64 elements in bfloat16 over 384 rows 6.2 / 8.2, 512
  // 6.9 / 8.2, 768 8.3 / 8.2; 4 heads of 128 in e4m3 over 256 8.1 / 9.8, 384 9.3 / 9.8, 512 10.5 / 9.9; 64 in float32
  // over 512 6.9 / 8.2, 768 8.6 / 8.1; 4 heads of 128 in float32 over 256 12.0 / 11.5, 384 15.7 / 11.5.  Many: 256 of 4
  // heads of 128 in e4m3 over 1000 18.1 / 23.9, up to 4000 45.8 / 40.1; 512 of them over 2000 44.9 / 54.4, up to 4000
  // 67.7 / 69.1, up to 8000 130 / 121; 512 of 64 in float32 over up to 4000 121 / 126, in int8 under float32 queries
  // over up to 2000 31 / 28, up to 4000 58 / 48.
  const long long most = units >= 512 ? (*mfma || !small ? 4096 : 2048)
                         : units >= 256 ? 1024
                         : *mfma        ? (small || D > 64 ? 384 : 512)
                                        : std::min(512, 512 * 64 / (p.heads * D));
  const bool one = T <= most;
  // Shares pay where a place gets many steps and the units' rows differ: 64 sequences of up to 8000, 8 heads of 64 in
  // bfloat16 110 us against 121 in chunks (equal ones 164 against 162), 8 of 128 in e4m3 121 against 123.  Not
  // over wide rows of 16 bits, whose registers they spill (the same of 128 in bfloat16, 8 heads each: 242 against
  // 239, equal ones 359 against 321).  One sequence's chunks are equal as they are.
  if (*mfma && !one && p.c.B > 1 && p.c.B <= kShareSeqs && paged_mfma_shares(cache_dtype, D) && steps >= 16 * places &&
      steps < (1ll << 30)) {
    p.shares = (int)places;
    return places + units;
  }
  // Rows of a chunk, a power of two: about as many workgroups as places on the chip, not so short that a
  // workgroup's beginning and end outweigh its rows.  Measured at 128 / 256 / 512 / 1024 / 2048 rows: one sequence
  // of 131072, 8 heads of 64: 50.5 / 47.7 / 46.3 / 46.0 / 46.2 us (1024 taken); 32 of up to 2048, 12 heads of
  // 64: - / 30.4 / 30.5 / 32.1 / 33.4 (512); 16 of up to 16001, one head of 96: 24.7 / 21.0 / 20.1 / 19.8 / 23.6
  // (256); 5 of up to 5001, 3 heads of 80 over int8: 13.2 / 13.6 / 16.4 / 22.2 / 35 (128).
  long long chunk = 128;
  while (chunk < (one ? T : 4096) && (one || chunk * 3 * places < T * units * 2)) chunk *= 2;
  while ((T + chunk - 1) / chunk > 65535) chunk *= 2;  // (the grid's limit)
  p.splits = (int)((T + chunk - 1) / chunk);
  p.chunk = (int)chunk;
  return p.splits > 1 ? units * p.splits : 0;
}

template <int QT, int CT, int D, int GT>
void launch(const PagedDecode& p, hipStream_t st) {
  const unsigned units = (unsigned)(p.c.B * p.c.Hkv * ((p.G + GT - 1) / GT));
  hipLaunchKernelGGL((paged_decode_kernel<QT, CT, D, GT>), dim3(units, (unsigned)p.splits), dim3(kBlock), 0, st, p);
}

template <int QT, int CT, int D>
void launch_heads(const PagedDecode& p, hipStream_t st) {
  if (p.heads == 1) {
    launch<QT, CT, D, 1>(p, st);
  } else if (p.heads == 2) {
    launch<QT, CT, D, 2>(p, st);
  } else if constexpr (RowMap<D>::pieces == 1) {
    launch<QT, CT, D, 4>(p, st);
  }
}

template <int QT, int D>
void launch_types(const PagedDecode& p, bool mfma, int ct, hipStream_t st) {
  if (mfma) launch_paged_mfma(p, QT, ct, D, st);
  else if (ct == DSQG_E4M3) launch_heads<QT, DSQG_E4M3, D>(p, st);
  else if (ct == DSQG_INT8) launch_heads<QT, DSQG_INT8, D>(p, st);
  else if constexpr (QT == DSQG_F32) launch_heads<QT, QT, D>(p, st);
  if (!p.joins) return;
  // The join's rows of lanes: about as many as a unit has parts; it takes any number.
  const long long blocks = units_of(p) * p.heads, parts = p.shares ? 2 + p.shares / units_of(p) : p.splits;
  hipLaunchKernelGGL((paged_join_kernel<QT, D>), dim3((unsigned)blocks), dim3(parts > 32 ? 1024 : parts > 4 ? 256 : 64), 0, st, p);
}

template <int QT>
void launch_dim(const PagedDecode& p, bool mfma, int ct, int D, hipStream_t st) {
  switch (D) {
    case 32: launch_types<QT, 32>(p, mfma, ct, st); break;
    case 64: launch_types<QT, 64>(p, mfma, ct, st); break;
    case 80: launch_types<QT, 80>(p, mfma, ct, st); break;
    case 96: launch_types<QT, 96>(p, mfma, ct, st); break;
    default: launch_types<QT, 128>(p, mfma, ct, st); break;
  }
}

// The checks that the size query and the launch share; workspace bytes of the parts.
int check_decode(const dsqg_paged_decode_args* a, PagedDecode* p, bool* mfma, long long* parts) {
  if (!a || a->H < 0) return DSQG_EINVAL;
  *p = PagedDecode{};
  *mfma = false;
  *parts = 0;
  if (const int st = check_paged_cache(a->cache, &p->c)) return st;
  const dsqg_paged_cache& c = a->cache;
  if (c.cache_dtype <= DSQG_F16 && c.cache_dtype != c.dtype) return DSQG_EINVAL;
  if (c.Hkv > 0 ? a->H == 0 || a->H % c.Hkv != 0 : a->H != 0) return DSQG_EINVAL;
  if ((long long)c.B * a->H == 0) return DSQG_OK;
  if ((long long)c.B * a->H >= (1ll << 21)) return DSQG_EUNSUPPORTED;  // grid: a join of 1024 for each, rounded up to units
  // Offsets inside a page, and from page to page, are 32 bits.
  if (p->c.kn * c.page >= (1ll << 31) || p->c.vn * c.page >= (1ll << 31) || p->c.kp >= (1ll << 31) || p->c.vp >= (1ll << 31))
    return DSQG_EUNSUPPORTED;
  p->H = a->H;
  p->G = a->H / c.Hkv;
  *parts = plan(*p, c.dtype, c.cache_dtype, c.D, mfma);
  return *parts < (1ll << 31) ? DSQG_OK : DSQG_EUNSUPPORTED;
}

// Bytes of the parts, D sums, a maximum and a sum for each head, and of the joins.
size_t part_bytes(const PagedDecode& p, long long parts, int D) {
  return parts ? (size_t)parts * p.heads * (D + 2) * sizeof(float) + (size_t)units_of(p) * sizeof(int2) : 0;
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" int dsqg_paged_decode_workspace_size(const dsqg_paged_decode_args* a, size_t* bytes) {
  PagedDecode p;
  bool mfma;
  long long parts;
  if (!bytes) return DSQG_EINVAL;
  if (const int st = check_decode(a, &p, &mfma, &parts)) return st;
  *bytes = part_bytes(p, parts, a->cache.D);
  return DSQG_OK;
}

extern "C" int dsqg_paged_decode(const dsqg_paged_decode_args* a, dsqg_stream_t stream) {
  PagedDecode p;
  bool mfma;
  long long parts;
  if (const int st = check_decode(a, &p, &mfma, &parts)) return st;
  const dsqg_paged_cache& c = a->cache;
  if ((long long)c.B * a->H == 0) return DSQG_OK;
  const long long es = elem_size(c.dtype);
  auto row = [&](const void* ptr, const int64_t st[2]) {
    if (!ptr || (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0) return false;
    for (int i = 0; i < 2; ++i)
      if (st[i] < 0 || st[i] > (1ll << 50) || st[i] * es % 16 != 0) return false;
    return true;
  };
  if (!row(a->q, a->q_stride) || !a->pos || !a->out || (reinterpret_cast<uintptr_t>(a->out) & 15u) != 0) return DSQG_EINVAL;
  if (!a->k_new != !a->v_new) return DSQG_EINVAL;
  if (a->k_new && (!row(a->k_new, a->k_new_stride) || !row(a->v_new, a->v_new_stride))) return DSQG_EINVAL;
  if (parts > 0) {
    if (!a->workspace || a->workspace_bytes < part_bytes(p, parts, c.D)) return DSQG_EWORKSPACE;
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return DSQG_EINVAL;
  }
  p.scale = a->softmax_scale * 1.4426950408889634f;
  p.q = static_cast<const char*>(a->q); p.qb = a->q_stride[0] * es; p.qh = a->q_stride[1] * es;
  p.kn = static_cast<const char*>(a->k_new); p.knb = a->k_new_stride[0] * es; p.knh = a->k_new_stride[1] * es;
  p.vn = static_cast<const char*>(a->v_new); p.vnb = a->v_new_stride[0] * es; p.vnh = a->v_new_stride[1] * es;
  p.pos = reinterpret_cast<const long long*>(a->pos);
  p.out = static_cast<char*>(a->out);
  if (parts > 0) {
    p.acc = static_cast<float*>(a->workspace);
    p.ml = p.acc + parts * p.heads * c.D;
    p.joins = reinterpret_cast<int2*>(p.ml + parts * p.heads * 2);
  }
  // Pools of more than a third of the 256 MB Infinity Cache are not found there by the next step, or only at
  // the cost of what else it holds: rows read past it take 10 % less time at 130 to 680 MB, but 11 to 14 % more
  // at 62 MB, which the cache serves.
  p.stream = 2ll * c.P * c.Hkv * c.page * c.D * elem_size(c.cache_dtype) > (85ll << 20);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (c.dtype == DSQG_F32) launch_dim<DSQG_F32>(p, mfma, c.cache_dtype, c.D, st);
  else if (c.dtype == DSQG_BF16) launch_dim<DSQG_BF16>(p, mfma, c.cache_dtype, c.D, st);
  else launch_dim<DSQG_F16>(p, mfma, c.cache_dtype, c.D, st);
  return hipGetLastError() == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
