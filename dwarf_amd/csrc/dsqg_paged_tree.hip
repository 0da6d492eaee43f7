// Steps of several tokens over a paged cache (gfx950): drafts as trees or chains, and single tokens of a windowed layer.
//
//   out_i = sum_t softmax_t(scale q_i . k_t) v_t     over the positions before the draft, node i's ancestors and itself,
//
// of those the ones within the window of node i's place (the draft's position plus its depth), and the sinks.
//
// The G query heads of a key/value head times the T nodes are the columns of S^T = K Q^T and O^T += V^T P^T, in groups of
// 16 NQ; a wave takes tiles of 32 positions, whose rows go from memory to operands as in dsqg_paged_mfma.hip, and
// serve all columns of its group.  float32 queries take the float32 matrix instructions (16x16x4), which round no
// product.  Rows of the draft are written to their pages first, by every workgroup that reads them (each writes the
// same bytes), so that a step attends what the cache will hold and needs no launch of its own for it.
//
// Masks are needed in few tiles: those that hold rows of the draft and, with a window, those where it begins and the sinks'.
// There a node's ancestors are one 64-bit word, found by doubling pointers over the wave (lane j: node j).  A value
// that some columns of such a tile do not see must not reach them, not even as 0 times an infinity: where a tile with
// masks holds infinities or NaN, its second product runs a column at a time, the other's values taken out.  8 bits have the NaN
// of e4m3 alone (which no writer here makes): a zero takes its place in the product, and the sums that see it are NaN in the end.
//
// Weights of groups of 16 columns enter the second product as two 16-bit terms (dsqg_paged_mfma.hip: 2^-16 of the weight),
// those of larger groups, which arithmetic bounds, as one: a rounding of up to 2^-8 (bfloat16) or 2^-11 (float16) of each
// weight, of the size of the output's own.  (float16 queries over 8-bit rows, whose operands are bfloat16: two again, for
// 2^-8 is more than their output's rounding.)  Scores, statistics and sums are fp32.
//
// Measured: 16 sequences of up to 8192, 8 key/value heads of 4, 64 nodes, D = 128 over e4m3, 309 us, 281 TFLOP/s: vector
// instructions (a weight's and the codes', of which 32 columns share each) and the latency of two waves a SIMD bound it.
// 32 sequences of up to 2048, 12 heads, 26 nodes, D = 64 in bfloat16, 42 us, 3.2 TB/s; one node within a window of 1024 of
// 8191, 25 us, 3.9 TB/s: reads of pages, each wave a tile ahead.  One sequence of 77 in float32, 8 us: a launch's latency.
#include <algorithm>

#include "dsqg_launch.hpp"
#include "dsqg_paged_tile.hpp"

namespace dsqg {
namespace {

typedef unsigned long long u64;

struct PagedTree {
  PagedCache c;
  int H, G, T;             // query heads, of one key/value head; nodes
  int cols;                // columns of a key/value head, T * G rounded up to its groups
  float scale;             // softmax_scale * log2(e)
  const char* q; long long qb, qh, qt;   // strides in bytes
  const char* kn; long long knb, knh, knt;
  const char* vn; long long vnb, vnh, vnt;
  const int* parents; long long ps;      // or null: a chain
  const long long* counts;               // or null
  const long long* pos;
  int window, sinks;       // window 0: none
  char* out;               // [B, T, H, D]
  int chunk, splits;       // tiles of a workgroup's part, and parts
  int stream;              // rows are read past the caches' retention
  int words;               // scale bytes lie so that four rows' are one word
  float* ml;               // workspace [B * Hkv, splits, cols, 2]
  float* acc;              // ... [B * Hkv, splits, cols, D]
};

// The tiles that a sequence's step reads: `sinks` of them from the beginning, then those from `from` on.
struct Span {
  int sinks, from, n;
  __device__ __forceinline__ int tile(int v) const { return v < sinks ? v : v - sinks + from; }
};

// Nodes of sequence b (0: none, also where it is not in use).
__device__ __forceinline__ int nodes_of(const PagedTree& p, int b, long long pos) {
  if (pos < 0) return 0;
  return p.counts ? (int)max(0ll, min((long long)p.T, load_const(p.counts + b))) : p.T;
}

__device__ __forceinline__ bool in_table(const PagedTree& p, long long pos) { return pos <= ((long long)p.c.M << p.c.shift); }

// pos is in the table, nodes > 0.
__device__ __forceinline__ Span span_of(const PagedTree& p, int pos, int nodes) {
  Span s = {0, 0, 0};
  if (p.window) {
    const int lo = max(0, pos - p.window + 1);
    s.sinks = (min(p.sinks, lo) + kTile - 1) / kTile;
    s.from = max(s.sinks, lo / kTile);
  }
  s.n = s.sinks + (pos + nodes + kTile - 1) / kTile - s.from;
  return s;
}

__device__ __forceinline__ int parts_of(const PagedTree& p, int n) { return (n + p.chunk - 1) / p.chunk; }

// Eight operand values.
template <bool FP32> struct Frag { uint4 x; };
template <> struct Frag<true> { float x[8]; };

template <bool FP32, bool F16>
__device__ __forceinline__ f32x4_t mma(const Frag<FP32>& a, const Frag<FP32>& b, f32x4_t c) {
  if constexpr (FP32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[e], b.x[e], c, 0, 0, 0);
    return c;
  } else {
    return mfma32<F16>(a.x, b.x, c);
  }
}

// Infinities and NaN among four words of a type's elements.
template <int CT>
__device__ __forceinline__ bool odd_values(uint4 v) {
  constexpr uint32_t e = CT == DSQG_F32 ? 0x7f800000u : CT == DSQG_BF16 ? 0x7f80u : 0x7c00u;
  bool odd = false;
  for (uint32_t w : {v.x, v.y, v.z, v.w}) {
    odd |= (w & e) == e;
    if constexpr (CT != DSQG_F32) odd |= (w & (e << 16)) == e << 16;
  }
  return odd;
}

// NaN among four e4m3 codes (0x7f with either sign): a byte's top bit is set where its other seven are, as one added to them carries.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Whether a group's queries are read from LDS for each tile, where they would take 32 registers of a wave or more.
constexpr bool queries_in_lds(int QT, int CT, int D, int NQ) {
  return QT != DSQG_F32 && !(QT == DSQG_F16 && narrow(CT)) && NQ * ((D + 31) / 32) >= 8;
}

template <int QT, int CT, int D, int NQ>
__global__ __launch_bounds__(kBlock, QT == DSQG_F32 ? 1 : 2) void paged_tree_kernel(PagedTree p) {
  using S = Steps<CT, D>;
  using V = ValueMap<CT, D>;
  constexpr bool FP32 = QT == DSQG_F32;
  constexpr bool F16 = CT == DSQG_F16;                // operands in float16 (else bf16, where they are 16 bits)
  constexpr bool QLO = QT == DSQG_F16 && narrow(CT);  // queries in two terms
  constexpr bool PLO = !FP32 && (NQ == 1 || QLO);     // weights in two terms
  constexpr int ES = elem_size(CT), KS = S::count, DB = D / 16;
  // Row stride of staged values, in elements: of 16 bits an odd multiple of eight banks, so that the transposed reads, of four
  // pieces of sixteen rows, meet in none.
  constexpr int RV = FP32 ? D + 4 : D % 32 == 0 ? D + 16 : D;
  typedef typename std::conditional<FP32, float, bf16_t>::type val_t;
  __shared__ __align__(16) val_t sV[kWaves][kTile * RV];
  __shared__ float wm[kWaves][16], wl[kWaves][16];
  // e4m3: which elements of a lane's sums see a NaN in a tile with masks.
  __shared__ uint32_t sees_nan[CT == DSQG_E4M3 ? kWaves : 1][NQ][64];
  static_assert(4 * DB <= 32, "a bit for each");
  constexpr bool QLDS = queries_in_lds(QT, CT, D, NQ);
  __shared__ uint4 sQ[QLDS ? NQ * KS : 1][QLDS ? 64 : 1];  // a lane's fragments

  const int groups = p.cols / (16 * NQ);
  const int unit = blockIdx.x;  // (grid.x is rounded up, so that a unit's groups run on one XCD)
  if (unit >= p.c.B * p.c.Hkv) return;
  const int b = unit / p.c.Hkv, hk = unit - b * p.c.Hkv;
  const int split = blockIdx.y / groups, c0 = (blockIdx.y - split * groups) * 16 * NQ;
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = l & 15, g = l >> 4;
  const int M = p.T * p.G;
  const long long pos64 = load_const(p.pos + b);
  const int nodes = nodes_of(p, b, pos64);
  const bool inside = in_table(p, pos64);
  auto out_at = [&](int m) {  // of column m
    const int t = m / p.G;
    return (((long long)b * p.T + t) * p.H + hk * p.G + (m - t * p.G)) * D;
  };
  if ((nodes == 0 || !inside) && split != 0) return;
  // Ancestors of node l, itself among them; none where its parents do not lead, each an earlier node, to -1.
  u64 above = 0, any = 0;
  int depth = 0;
  {
    int to = -2;
    if (l < nodes) {
      const int parent = p.parents ? p.parents[b * p.ps + l] : l - 1;
      to = parent >= -1 && parent < l ? parent : -2;
    }
    above = l < nodes ? 1ull << l : 0;
#pragma unroll
    for (int r = 0; r < 6; ++r) {
      const u64 x = __shfl(above, max(to, 0), 64);
      const int y = __shfl(to, max(to, 0), 64);
      if (to >= 0) {
        above |= x;
        to = y;
      }
    }
    if (to != -1) above = 0;
    depth = __popcll(above) - 1;
    if (p.window && above) {
      // (Ancestors are at the places pos, pos + 1, .. on the way down.)
      u64 rest = above;
      for (int d = 0; rest; ++d) {
        const u64 bit = rest & -rest;
        rest &= rest - 1;
        if (d <= depth - p.window && pos64 + d >= p.sinks) above &= ~bit;
      }
    }
    any = above;
#pragma unroll
    for (int o = 32; o; o >>= 1) any |= __shfl_xor(any, o, 64);
  }
  // ... and of this lane's columns.
  u64 sees[NQ];
  int lo[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int m = c0 + 16 * n + i, t = m / p.G;
    sees[n] = __shfl(above, t & 63, 64);
    const int d = __shfl(depth, t & 63, 64);
    if (m >= M) sees[n] = 0;
    lo[n] = p.window && inside ? max(0, (int)pos64 + d - p.window + 1) : 0;
  }
  if (nodes == 0 || !inside) {  // no nodes: zeros; past the table: NaN
    if (wave == 0) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int m = c0 + 16 * n + i;
        if (m < M)
          for (int d = g; d < D; d += 4) store_out<QT>(p.out, out_at(m) + d, sees[n] ? __uint_as_float(0x7fc00000u) : 0.f);
      }
    }
    return;
  }
  const int pos = (int)pos64;
  const Span span = span_of(p, pos, nodes);
  const int count = parts_of(p, span.n);
  if (split >= count) return;
  const int v0 = split * p.chunk, v1 = min(span.n, v0 + p.chunk);

  // Rows of the draft to their pages, where this part reads any.
  if (p.kn && span.tile(v1 - 1) * kTile + kTile > pos) {
    using R = RowMap<D>;
    const int rg = threadIdx.x % R::lanes;
    for (int n = threadIdx.x / R::lanes; n < nodes; n += kBlock / R::lanes) {
      const int t = pos + n;
      const int page = (t >> p.c.shift) < p.c.M ? p.c.table[b * p.c.ts + (t >> p.c.shift)] : -1;
      if ((unsigned)page >= (unsigned)p.c.P) continue;
      const long long slot = t & ((1 << p.c.shift) - 1);
      Raw8<QT> x[R::pieces], y[R::pieces];
#pragma unroll
      for (int u = 0; u < R::pieces; ++u) {
        raw_zero<QT>(x[u]);
        raw_zero<QT>(y[u]);
        if (rg + R::lanes * u < R::CPR) {
          x[u] = raw_load<QT>(p.kn + b * p.knb + hk * p.knh + n * p.knt + (rg + R::lanes * u) * 8 * elem_size(QT));
          y[u] = raw_load<QT>(p.vn + b * p.vnb + hk * p.vnh + n * p.vnt + (rg + R::lanes * u) * 8 * elem_size(QT));
        }
      }
      put_row<QT, CT, D>(p.c.k + page * p.c.kp + hk * p.c.kh + slot * p.c.kn,
                         p.c.ks + page * p.c.ksp + hk * p.c.ksh + slot * p.c.ksn, x, rg);
      put_row<QT, CT, D>(p.c.v + page * p.c.vp + hk * p.c.vh + slot * p.c.vn,
                         p.c.vs + page * p.c.vsp + hk * p.c.vsh + slot * p.c.vsn, y, rg);
    }
    __syncthreads();  // (they come back through the same CU's L1, which the stores went through)
  }

  // Tiles from all_from on that end before the draft have no masks; rows below any_from that are no sinks are seen by nobody.
  const int all_from = p.window ? max(0, pos + nodes - p.window) : 0, any_from = p.window ? max(0, pos - p.window + 1) : 0;

  Frag<FP32> qh[QLDS ? 1 : NQ][KS], ql[NQ][QLO ? KS : 1];
  if constexpr (QLDS) {
    for (int e = wave; e < NQ * KS; e += kWaves) {
      const int n = e / KS, m = c0 + 16 * n + i, t = m / p.G, d = S::at(e - n * KS, g);
      Raw8<QT> r;
      raw_zero<QT>(r);
      if (m < M && d < D) r = raw_load<QT>(p.q + b * p.qb + (hk * p.G + m - t * p.G) * p.qh + t * p.qt + d * elem_size(QT));
      sQ[e][l] = r.a;
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < (QLDS ? 0 : NQ); ++n) {
    const int m = c0 + 16 * n + i, t = m / p.G;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Raw8<QT> r;
      raw_zero<QT>(r);
      const int d = S::at(s, g);
      if (m < M && d < D) r = raw_load<QT>(p.q + b * p.qb + (hk * p.G + m - t * p.G) * p.qh + t * p.qt + d * elem_size(QT));
      if constexpr (FP32) {
        raw_floats<QT>(r, qh[n][s].x);
      } else if constexpr (QLO) {
        float x[8];
        raw_floats<QT>(r, x);
        split8(x, qh[n][s].x, ql[n][s].x);
      } else {
        qh[n][s].x = r.a;
      }
    }
  }

  // The wave's tile, as in dsqg_paged_mfma.hip.
  Raw8<CT> kr[2][KS];
  uint4 vr[V::passes][V::per_lane];
  uint32_t eks[2] = {}, evs[2] = {};
  bool bad[2];
  const int kn = (int)p.c.kn, vn = (int)p.c.vn;
  const int klane = i * kn + g * (narrow(CT) && S::pairs > 0 ? 16 : 8 * ES);
  const int krest = i * kn + 8 * ES * g;  // the steps behind the pairs
  const int vlane = (l / V::lanes & 15) * vn + l % V::lanes * 16;
  val_t* const sVw = sV[wave];
  const long long kh = hk * p.c.kh, vh = hk * p.c.vh, ksh = hk * p.c.ksh, vsh = hk * p.c.vsh;
  const int* table = p.c.table + b * p.c.ts;
  const int first = v0 + wave;
  // Page numbers of the wave's next 32 tiles, one half each lane.
  auto pages_from = [&](int v) {
    const int t = span.tile(v + (l >> 1) * kWaves) * kTile + 16 * (l & 1);
    return (t >> p.c.shift) < p.c.M ? table[t >> p.c.shift] : -1;
  };
  int pages = pages_from(first);

  auto load_as = [&](int k, auto aux) {  // the wave's tile k; aux: the loads' cache policy
    constexpr int AUX = decltype(aux)::value;
    if ((k & 31) == 0 && k > 0) pages = pages_from(first + k * kWaves);
    const int tile = span.tile(first + k * kWaves) * kTile;
    __amdgpu_buffer_rsrc_t rk[2], rv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int page = __builtin_amdgcn_readlane(pages, 2 * (k & 31) + h);
      bad[h] = (unsigned)page >= (unsigned)p.c.P;
      const unsigned at = bad[h] ? 0u : (unsigned)page;
      const unsigned slot = (unsigned)(tile + 16 * h) & ((1u << p.c.shift) - 1u);
      auto rows = [&](char* base, long long page_stride, int row_stride, long long head) {
        return __builtin_amdgcn_make_buffer_rsrc(
            base + (u64)at * (unsigned)page_stride + slot * (unsigned)row_stride + head, (short)0, 15 * row_stride + D * ES,
            0x00020000);
      };
      rk[h] = rows(p.c.k, p.c.kp, kn, kh);
      rv[h] = rows(p.c.v, p.c.vp, vn, vh);
      if constexpr (narrow(CT)) {
        auto bytes = [&](const unsigned char* base, long long page_stride, long long head, long long row_stride) {
          const unsigned char* s = base + at * page_stride + head + (slot + 4 * g) * row_stride;
          if (p.words) return *reinterpret_cast<const uint32_t*>(s);
          return s[0] | (uint32_t)s[row_stride] << 8 | (uint32_t)s[2 * row_stride] << 16 | (uint32_t)s[3 * row_stride] << 24;
        };
        eks[h] = bytes(p.c.ks, p.c.ksp, ksh, p.c.ksn);
        evs[h] = bytes(p.c.vs, p.c.vsp, vsh, p.c.vsn);
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
        const int off = krest + S::at(s, 0) * ES;
        if constexpr (narrow(CT)) {
          kr[h][s].a = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rk[h], off, 0, AUX));
        } else {
          kr[h][s].a = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk[h], off, 0, AUX));
          if constexpr (CT == DSQG_F32) kr[h][s].b = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk[h], off + 16, 0, AUX));
        }
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

  // Whether a row is seen by any node, and by one that sees `mask` of the draft and stored rows from `from` on.
  auto seen_by = [&](int t, u64 mask, int from) __attribute__((always_inline)) {
    const int j = t - pos;
    return j < 0 ? t >= from || t < p.sinks : j < 64 && ((mask >> j) & 1);
  };

  // e4m3: marks for the sums that see a NaN among the tile's staged rows, and zeros in its place.  (Inlined by force, as what it is
  // called from: out of line, the arrays that these refer to are memory, and the whole kernel takes twice its time.)
  auto nan_at = [&](int row, int d) __attribute__((always_inline)) {  // of elements 16 d + 4 g on, which this lane sums
    const val_t* const x = sVw + row * RV + 16 * d + 4 * g;
    uint32_t in = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (FP32) in |= (x[e] != x[e] ? 1u : 0u) << e;
      else in |= ((x[e] & 0x7fff) > 0x7f80 ? 1u : 0u) << e;
    }
    return in;
  };
  auto take_nan = [&](int tile) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const u64 mask = sees[n];
      const int from = lo[n];
      uint32_t in = sees_nan[wave][n][l];
#pragma unroll 1
      for (int at = 0; at < kTile * DB; ++at)
        if (seen_by(tile + at / DB, mask, from)) in |= nan_at(at / DB, at % DB) << (4 * (at % DB));
      sees_nan[wave][n][l] = in;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int at = 0; at < kTile * DB; ++at) {
      const uint32_t in = nan_at(at / DB, at % DB);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((in >> e) & 1) sVw[at / DB * RV + 16 * (at % DB) + 4 * g + e] = 0;  // (the lanes of a group write the same)
    }
  };

  // The tile's value rows to LDS as operand values, zeros in the place of those that nobody sees; says whether an
  // infinity or NaN is among the others of a tile with masks.
  auto stage = [&](int tile, bool masks) __attribute__((always_inline)) {
    bool odd = false;
    if constexpr (CT == DSQG_E4M3) {
      if (masks) {
        asm volatile("");  // (a branch)
        uint32_t any_nan = 0;
#pragma unroll
        for (int u = 0; u < V::passes; ++u)
#pragma unroll
          for (int w = 0; w < V::per_lane; ++w)
            any_nan |= nan_codes(vr[u][w].x) | nan_codes(vr[u][w].y) | nan_codes(vr[u][w].z) | nan_codes(vr[u][w].w);
        odd = any_nan != 0;
      }
    }
#pragma unroll
    for (int u = 0; u < V::passes; ++u) {
      const int row = u * V::rows + l / V::lanes;
      // (An AND of every word: the compiler lost the first one of a choice between two uint4.)
      const uint32_t keep = !masks || seen_by(tile + row, any, any_from) ? ~0u : 0u;
#pragma unroll
      for (int w = 0; w < V::per_lane; ++w) {
        const int piece = l % V::lanes + V::lanes * w;
        const uint4 x = make_uint4(vr[u][w].x & keep, vr[u][w].y & keep, vr[u][w].z & keep, vr[u][w].w & keep);
        if (piece < V::pieces) {
          if constexpr (narrow(CT)) {
            Raw8<CT> part[2];
            part[0].a = make_uint2(x.x, x.y);
            part[1].a = make_uint2(x.z, x.w);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if constexpr (FP32) {
                float f[8];
                raw_floats<CT>(part[h], f);
                *reinterpret_cast<float4*>(sVw + row * RV + 16 * piece + 8 * h) = make_float4(f[0], f[1], f[2], f[3]);
                *reinterpret_cast<float4*>(sVw + row * RV + 16 * piece + 8 * h + 4) = make_float4(f[4], f[5], f[6], f[7]);
              } else {
                st16(sVw + row * RV + 16 * piece + 8 * h, operand<CT>(part[h]));
              }
            }
          } else {
            if (masks) odd |= odd_values<CT>(x);
            st16(reinterpret_cast<char*>(sVw) + (row * RV) * (int)sizeof(val_t) + 16 * piece, x);
          }
        }
      }
    }
    odd = masks && __any(odd);
    if constexpr (CT == DSQG_E4M3)
      if (__builtin_expect(odd, 0)) take_nan(tile);
    return odd;
  };

  float m[NQ], lsum[NQ];  // the weights' reference exponent, the sum over this lane's rows
  f32x4_t o[NQ][DB];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = -INFINITY;
    lsum[n] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[n][d] = zero4();
  }
  const float nan = __uint_as_float(0x7fc00000u);
  if constexpr (CT == DSQG_E4M3) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) sees_nan[wave][n][l] = 0;
  }

  if (first < v1) load(0);
#pragma unroll 1
  for (int k = 0, v = first; v < v1; ++k, v += kWaves) {
    const int tile = span.tile(v) * kTile;
    const bool masks = tile + kTile > pos || tile < all_from;
    f32x4_t s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = zero4();
    if constexpr (QLDS) {
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        Frag<FP32> a[2], q;
#pragma unroll
        for (int h = 0; h < 2; ++h) a[h].x = operand<CT>(kr[h][e]);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          q.x = sQ[n * KS + e][l];
#pragma unroll
          for (int h = 0; h < 2; ++h) s[n][h] = mma<FP32, F16>(a[h], q, s[n][h]);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < KS; ++e) {
          Frag<FP32> a;
          if constexpr (FP32) raw_floats<CT>(kr[h][e], a.x);
          else a.x = operand<CT>(kr[h][e]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            s[n][h] = mma<FP32, F16>(a, qh[n][e], s[n][h]);
            if constexpr (QLO) s[n][h] = mma<FP32, F16>(a, ql[n][e], s[n][h]);
          }
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
    const bool odd_rows = stage(tile, masks);
    const uint32_t ek[2] = {eks[0], eks[1]}, ev[2] = {evs[0], evs[1]};
    const bool no[2] = {bad[0], bad[1]};
    // The next tile's rows are on their way during the softmax and the second product.
    if (v + kWaves < v1) load(k + 1);
    __builtin_amdgcn_sched_barrier(0);

    Frag<FP32> wh[NQ], wlo[PLO ? NQ : 1];
    bool odd = false;
    if constexpr (narrow(CT))
      odd = __any((((0xfefefefeu - ek[0]) & ek[0]) | ((0xfefefefeu - ek[1]) & ek[1]) | ((0xfefefefeu - ev[0]) & ev[0]) |
                   ((0xfefefefeu - ev[1]) & ev[1])) & 0x80808080u);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float x[8], w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = s[n][e / 4][e % 4] * p.scale;
        if constexpr (narrow(CT)) x[e] = __builtin_amdgcn_ldexpf(x[e], (int)((ek[e / 4] >> (8 * (e % 4))) & 255) - 127);
      }
      if (__builtin_expect(odd | no[0] | no[1], 0)) {
        asm volatile("");  // (a branch)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (no[e / 4] || (narrow(CT) && ((ek[e / 4] >> (8 * (e % 4))) & 255) == 255)) x[e] = nan;
      }
      uint32_t hide = 0;
      if (masks) {
        asm volatile("");
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool hidden = !seen_by(tile + 16 * (e / 4) + 4 * g + e % 4, sees[n], lo[n]);
          hide |= (hidden ? 1u : 0u) << e;
          x[e] = hidden ? -INFINITY : x[e];
        }
      }
      float mx = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
      mx = col_max(mx);
      // (Where a score's step is 8 and more the lift may come out as 16, and a weight as 2^16, which is no single float16 number:
      // huge scores have no lift.)
      mx = F16 && !PLO && fabsf(mx) >= 65536.f ? mx : lifted<F16>(mx);
      if (__any(mx > m[n])) {
        const float mn = fmaxf(m[n], mx), a = weight(m[n], mn);
        m[n] = mn;
        lsum[n] *= a;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[n][d] *= a;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = weight(x[e], m[n]);
#pragma unroll
      for (int e = 0; e < 8; ++e) lsum[n] += w[e];
      if constexpr (narrow(CT)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_ldexpf(w[e], (int)((ev[e / 4] >> (8 * (e % 4))) & 255) - 127);
        if (__builtin_expect(odd, 0)) {
          asm volatile("");
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (((ev[e / 4] >> (8 * (e % 4))) & 255) == 255) w[e] = nan;
            if ((hide >> e) & 1) w[e] = 0.f;  // (a scale of a row that is not seen is no number of this column)
          }
        }
      }
      if constexpr (FP32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) wh[n].x[e] = w[e];
      } else if constexpr (PLO) {
        split_weights<F16, !narrow(CT)>(w, wh[n].x, wlo[n].x);
      } else if constexpr (F16) {
        // (A weight above zero stays so: an infinity times it is one.)
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = fmaxf(w[2 * e], fminf(w[2 * e] * 0x1p126f, 0x1p-24f));
          const float c = fmaxf(w[2 * e + 1], fminf(w[2 * e + 1] * 0x1p126f, 0x1p-24f));
          h[e] = __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)a, (_Float16)c});
        }
        wh[n].x = make_uint4(h[0], h[1], h[2], h[3]);
      } else {
        wh[n].x = make_uint4(cvt_pk_bf16(w[0], w[1]), cvt_pk_bf16(w[2], w[3]), cvt_pk_bf16(w[4], w[5]), cvt_pk_bf16(w[6], w[7]));
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the rows are staged
    __builtin_amdgcn_wave_barrier();
    auto values = [&](int d) {
      Frag<FP32> f;
      if constexpr (FP32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f.x[e] = sVw[(16 * (e / 4) + 4 * g + e % 4) * RV + 16 * d + i];
      } else {
        const bf16_t* vtr = sVw + (4 * g + (i >> 2)) * RV + 4 * (i & 3);
        const uint2 a = __builtin_bit_cast(uint2, lds_read_tr16(vtr + 16 * d));
        const uint2 c = __builtin_bit_cast(uint2, lds_read_tr16(vtr + 16 * RV + 16 * d));
        f.x = make_uint4(a.x, a.y, c.x, c.y);
      }
      return f;
    };
    if (narrow(CT) || !odd_rows) {
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const Frag<FP32> x = values(d);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          o[n][d] = mma<FP32, F16>(x, wh[n], o[n][d]);
          if constexpr (PLO) o[n][d] = mma<FP32, F16>(x, wlo[n], o[n][d]);
        }
        if (d % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll 1
        for (int c = 0; c < 16; ++c) {
          const u64 mask = __shfl(sees[n], c, 64);
          const int from = __shfl(lo[n], c, 64);
          bool keep[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) keep[e] = seen_by(tile + 16 * (e / 4) + 4 * g + e % 4, mask, from);
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            Frag<FP32> x = values(d);
            if constexpr (FP32) {
#pragma unroll
              for (int e = 0; e < 8; ++e) x.x[e] = keep[e] ? x.x[e] : 0.f;
            } else {
              auto half = [&](int e) { return (keep[e] ? 0xffffu : 0u) | (keep[e + 1] ? 0xffff0000u : 0u); };
              x.x = make_uint4(x.x.x & half(0), x.x.y & half(2), x.x.z & half(4), x.x.w & half(6));
            }
            f32x4_t y = mma<FP32, F16>(x, wh[n], zero4());
            if constexpr (PLO) y = mma<FP32, F16>(x, wlo[n], y);
            if (i == c) o[n][d] += y;
          }
        }
      }
    }
  }

  if constexpr (CT == DSQG_E4M3) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const uint32_t in = sees_nan[wave][n][l];
      if (!__any(in != 0)) continue;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][d][e] += (in >> (4 * d + e)) & 1 ? nan : 0.f;
    }
  }

  // The waves' parts meet in LDS, each in its own block, 16 columns at a time.
  static_assert(16 * D * 4 <= kTile * RV * (int)sizeof(val_t), "a wave's part fits its block");
  float* const sums = reinterpret_cast<float*>(sVw);  // [16][D]
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    if (n > 0) __syncthreads();
    const float total = col_sum(lsum[n]);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4_t*>(sums + i * D + 16 * d + 4 * g) = o[n][d];
    if (g == 0) {
      // (A column that is no node: nothing, whatever the tiles without masks gave it.)
      wm[wave][i] = sees[n] ? m[n] : -INFINITY;
      wl[wave][i] = sees[n] ? total : 0.f;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * D; e += kBlock) {
      const int h = e / D, d = e - h * D, col = c0 + 16 * n + h;
      if (col >= M) break;
      float mm = -INFINITY, ll = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, wm[w][h]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float a = weight(wm[w][h], mm);
        ll = fmaf(wl[w][h], a, ll);
        // (A wave that saw nothing of this column may hold anything.)
        x = wl[w][h] == 0.f ? x : fmaf(reinterpret_cast<const float*>(sV[w])[e], a, x);
      }
      if (count == 1) {
        store_out<QT>(p.out, out_at(col) + d, ll == 0.f ? 0.f : x / ll);
      } else {
        const long long at = ((long long)unit * p.splits + split) * p.cols + col;
        p.acc[at * D + d] = x;
        if (d == 0) {
          p.ml[2 * at] = mm;
          p.ml[2 * at + 1] = ll;
        }
      }
    }
  }
}

// Joins a column's parts.  Grid: [units * T * G].  A part is JL lanes of four elements; the workgroup's rows of lanes take
// parts in turn and meet in LDS: the order is fixed by the sequences' lengths.
template <int QT, int D>
__global__ __launch_bounds__(256) void tree_join_kernel(PagedTree p) {
  constexpr int JL = D <= 32 ? 8 : D <= 64 ? 16 : 32;
  const int M = p.T * p.G;
  const int unit = blockIdx.x / M, col = blockIdx.x - unit * M, rows = blockDim.x / JL;
  const int gl = threadIdx.x % JL, r = threadIdx.x / JL;
  const int b = unit / p.c.Hkv, hk = unit - b * p.c.Hkv;
  const long long pos = load_const(p.pos + b);
  const int nodes = nodes_of(p, b, pos);
  if (nodes == 0 || !in_table(p, pos)) return;
  const int parts = parts_of(p, span_of(p, (int)pos, nodes).n);
  if (parts == 1) return;  // (written by its only workgroup)
  const long long at0 = (long long)unit * p.splits * p.cols + col;
  float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = r; c < parts; c += rows) {
    const long long at = at0 + (long long)c * p.cols;
    const float2 s = *reinterpret_cast<const float2*>(p.ml + 2 * at);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (4 * gl < D) v = *reinterpret_cast<const float4*>(p.acc + at * D + 4 * gl);
    const float mn = fmaxf(m, s.x), a = weight(m, mn), w = weight(s.x, mn);
    m = mn;
    l = fmaf(l, a, s.y * w);
    x[0] = fmaf(x[0], a, v.x * w);
    x[1] = fmaf(x[1], a, v.y * w);
    x[2] = fmaf(x[2], a, v.z * w);
    x[3] = fmaf(x[3], a, v.w * w);
  }
  __shared__ float jm[256 / JL], jl[256 / JL], jx[256 / JL][D];
  if (4 * gl < D)
#pragma unroll
    for (int e = 0; e < 4; ++e) jx[r][4 * gl + e] = x[e];
  if (gl == 0) {
    jm[r] = m;
    jl[r] = l;
  }
  __syncthreads();
  const int n = min(rows, parts);
  m = -INFINITY;
  for (int e = 0; e < n; ++e) m = fmaxf(m, jm[e]);
  const int t = col / p.G;
  const long long out = (((long long)b * p.T + t) * p.H + hk * p.G + (col - t * p.G)) * D;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float s = 0.f;
    l = 0.f;
    for (int e = 0; e < n; ++e) {
      const float w = weight(jm[e], m);
      l = fmaf(jl[e], w, l);
      s = fmaf(jx[e][d], w, s);
    }
    store_out<QT>(p.out, out + d, l == 0.f ? 0.f : s / l);
  }
}

// Columns of a workgroup: 16 for each tile of the products.  Larger groups read the cache less often, and take more
// registers: four tiles where a wave's rows on their way and its sums leave room, those of 8-bit caches of up to 96 elements,
// else two, and two where queries have two terms or are float32.  (16 sequences of up to 8192, 8 key/value heads, 256 columns,
// e4m3: four 183 us and two 194 at D = 64, 214 and 265 at 80, 214 and 260 at 96, 364 and 331 at 128; bfloat16 at 64 either 120.)
constexpr bool four_tiles(int dtype, int cache_dtype, int D) { return dtype == DSQG_BF16 && narrow(cache_dtype) && D <= 96; }

int group_tiles(int M, int dtype, int cache_dtype, int D) {
  return M <= 16 ? 1 : M <= 32 || !four_tiles(dtype, cache_dtype, D) ? 2 : 4;
}

long long units_of(const PagedTree& p) { return (long long)p.c.B * p.c.Hkv; }

// Chooses the columns' groups and the split; returns the parts that may have to be joined.
long long plan(PagedTree& p, int dtype, int cache_dtype, int D) {
  const int M = p.T * p.G, wide = 16 * group_tiles(M, dtype, cache_dtype, D);
  p.cols = (M + wide - 1) / wide * wide;
  const long long units = units_of(p), groups = p.cols / wide;
  // The most tiles that a sequence of this table can have.
  long long rows = ((long long)p.c.M << p.c.shift) + p.T;
  if (p.window) rows = std::min(rows, (long long)p.window + p.T + 64 + (p.sinks + 31ll) / 32 * 32);
  const long long tiles = (rows + kTile - 1) / kTile;
  // Parts of two rounds of the waves at least, and as many as give each CU one: the join of more costs what their balance
  // gives (32 sequences of up to 2048, 12 heads, 26 nodes: 384 parts 42.5 us, 768 and their join 48; 77 tokens: 1 part 8.3 us, 2
  // and theirs 11).
  long long chunk = 8;
  while (chunk < tiles && chunk * 256 < tiles * units * groups) chunk *= 2;
  while ((tiles + chunk - 1) / chunk * groups > 65535) chunk *= 2;  // (the grid's limit)
  // Parts alike, of whole rounds of the waves.
  const long long parts = (tiles + chunk - 1) / chunk;
  chunk = ((tiles + parts - 1) / parts + kWaves - 1) / kWaves * kWaves;
  p.chunk = (int)chunk;
  p.splits = (int)((tiles + chunk - 1) / chunk);
  return p.splits > 1 ? units * p.splits * p.cols : 0;
}

template <int QT, int CT, int D, int NQ>
void launch(const PagedTree& p, hipStream_t st) {
  const unsigned units = (unsigned)((units_of(p) + 7) / 8 * 8);
  hipLaunchKernelGGL((paged_tree_kernel<QT, CT, D, NQ>), dim3(units, (unsigned)(p.splits * (p.cols / (16 * NQ)))), dim3(kBlock), 0, st, p);
}

template <int QT, int CT, int D>
void launch_groups(const PagedTree& p, int ct, hipStream_t st) {
  const int nq = group_tiles(p.T * p.G, QT, ct, D);
  if (nq == 1) return launch<QT, CT, D, 1>(p, st);
  if constexpr (four_tiles(QT, CT, D))
    if (nq == 4) return launch<QT, CT, D, 4>(p, st);
  launch<QT, CT, D, 2>(p, st);
}

template <int QT, int D>
void launch_types(const PagedTree& p, int ct, hipStream_t st) {
  if (ct == DSQG_E4M3) launch_groups<QT, DSQG_E4M3, D>(p, ct, st);
  else if (ct == DSQG_INT8) launch_groups<QT, DSQG_INT8, D>(p, ct, st);
  else launch_groups<QT, QT, D>(p, ct, st);
  if (p.splits == 1) return;
  hipLaunchKernelGGL((tree_join_kernel<QT, D>), dim3((unsigned)(units_of(p) * p.T * p.G)), dim3(p.splits > 4 ? 256 : 64), 0, st, p);
}

template <int QT>
void launch_dim(const PagedTree& p, int ct, int D, hipStream_t st) {
  switch (D) {
    case 32: launch_types<QT, 32>(p, ct, st); break;
    case 64: launch_types<QT, 64>(p, ct, st); break;
    case 80: launch_types<QT, 80>(p, ct, st); break;
    case 96: launch_types<QT, 96>(p, ct, st); break;
    default: launch_types<QT, 128>(p, ct, st); break;
  }
}

// The checks that the size query and the launch share, and the parts.
int check_tree(const dsqg_paged_tree_args* a, PagedTree* p, long long* parts) {
  if (!a || a->H < 0 || a->T < 1 || a->window < 0 || a->sinks < 0) return DSQG_EINVAL;
  *p = PagedTree{};
  *parts = 0;
  if (const int st = check_paged_cache(a->cache, &p->c)) return st;
  const dsqg_paged_cache& c = a->cache;
  if (c.cache_dtype <= DSQG_F16 && c.cache_dtype != c.dtype) return DSQG_EINVAL;
  if (c.Hkv > 0 ? a->H == 0 || a->H % c.Hkv != 0 : a->H != 0) return DSQG_EINVAL;
  if (a->T > DSQG_MAX_TREE) return DSQG_EUNSUPPORTED;
  if ((long long)c.B * a->H == 0) return DSQG_OK;
  // (The grid has less than 2^32 lanes in x.  The join's does: parts are for less than 256 groups of columns in all.)
  if ((long long)c.B * a->H * a->T >= (1ll << 30) || (long long)c.B * c.Hkv >= (1ll << 24) - 8) return DSQG_EUNSUPPORTED;
  // Offsets inside a page, and from page to page, are 32 bits.
  if (p->c.kn * c.page >= (1ll << 31) || p->c.vn * c.page >= (1ll << 31) || p->c.kp >= (1ll << 31) || p->c.vp >= (1ll << 31))
    return DSQG_EUNSUPPORTED;
  p->H = a->H;
  p->G = a->H / c.Hkv;
  p->T = a->T;
  // (No place is 2^30 positions from another, as none is that far from the first.)
  p->window = std::min(a->window, 1 << 30);
  p->sinks = p->window ? std::min(a->sinks, 1 << 30) : 0;
  const int wide = 16 * group_tiles(p->T * p->G, c.dtype, c.cache_dtype, c.D);
  if ((p->T * p->G + wide - 1) / wide > 65535) return DSQG_EUNSUPPORTED;  // (the grid in y, with a part for each)
  *parts = plan(*p, c.dtype, c.cache_dtype, c.D);
  return *parts < (1ll << 31) ? DSQG_OK : DSQG_EUNSUPPORTED;
}

size_t part_bytes(long long parts, int D) { return (size_t)parts * (D + 2) * sizeof(float); }

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" int dsqg_paged_tree_workspace_size(const dsqg_paged_tree_args* a, size_t* bytes) {
  PagedTree p;
  long long parts;
  if (!bytes) return DSQG_EINVAL;
  if (const int st = check_tree(a, &p, &parts)) return st;
  *bytes = part_bytes(parts, a->cache.D);
  return DSQG_OK;
}

extern "C" int dsqg_paged_tree(const dsqg_paged_tree_args* a, dsqg_stream_t stream) {
  PagedTree p;
  long long parts;
  if (const int st = check_tree(a, &p, &parts)) return st;
  const dsqg_paged_cache& c = a->cache;
  if ((long long)c.B * a->H == 0) return DSQG_OK;
  const long long es = elem_size(c.dtype);
  auto rows = [&](const void* ptr, const int64_t st[3]) {
    if (!ptr || (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0) return false;
    for (int i = 0; i < 3; ++i)
      if (st[i] < 0 || st[i] > (1ll << 50) || st[i] * es % 16 != 0) return false;
    return true;
  };
  if (!rows(a->q, a->q_stride) || !a->pos || !a->out || (reinterpret_cast<uintptr_t>(a->out) & 15u) != 0) return DSQG_EINVAL;
  if (!a->k_new != !a->v_new) return DSQG_EINVAL;
  if (a->k_new && (!rows(a->k_new, a->k_new_stride) || !rows(a->v_new, a->v_new_stride))) return DSQG_EINVAL;
  if (a->parents && (a->parents_stride < 0 || a->parents_stride > (1ll << 50))) return DSQG_EINVAL;
  if (parts > 0) {
    if (!a->workspace || a->workspace_bytes < part_bytes(parts, c.D)) return DSQG_EWORKSPACE;
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return DSQG_EINVAL;
  }
  p.scale = a->softmax_scale * 1.4426950408889634f;
  p.q = static_cast<const char*>(a->q);
  p.qb = a->q_stride[0] * es; p.qh = a->q_stride[1] * es; p.qt = a->q_stride[2] * es;
  p.kn = static_cast<const char*>(a->k_new);
  p.knb = a->k_new_stride[0] * es; p.knh = a->k_new_stride[1] * es; p.knt = a->k_new_stride[2] * es;
  p.vn = static_cast<const char*>(a->v_new);
  p.vnb = a->v_new_stride[0] * es; p.vnh = a->v_new_stride[1] * es; p.vnt = a->v_new_stride[2] * es;
  p.parents = a->parents;
  p.ps = a->parents_stride;
  p.counts = reinterpret_cast<const long long*>(a->counts);
  p.pos = reinterpret_cast<const long long*>(a->pos);
  p.out = static_cast<char*>(a->out);
  if (parts > 0) {
    p.acc = static_cast<float*>(a->workspace);
    p.ml = p.acc + parts * c.D;
  }
  const long long odd = p.c.ksp | p.c.ksh | p.c.vsp | p.c.vsh | (long long)reinterpret_cast<uintptr_t>(p.c.ks) |
                        (long long)reinterpret_cast<uintptr_t>(p.c.vs);
  p.words = narrow(c.cache_dtype) && p.c.ksn == 1 && p.c.vsn == 1 && odd % 4 == 0;
  // (As the single-token step's: pools larger than a third of the Infinity Cache.  Groups of columns find each other's
  // rows in L2 only if they stay there.)
  p.stream = p.cols == 16 * group_tiles(p.T * p.G, c.dtype, c.cache_dtype, c.D) &&
             2ll * c.P * c.Hkv * c.page * c.D * elem_size(c.cache_dtype) > (85ll << 20);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (c.dtype == DSQG_F32) launch_dim<DSQG_F32>(p, c.cache_dtype, c.D, st);
  else if (c.dtype == DSQG_BF16) launch_dim<DSQG_BF16>(p, c.cache_dtype, c.D, st);
  else launch_dim<DSQG_F16>(p, c.cache_dtype, c.D, st);
  return hipGetLastError() == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
