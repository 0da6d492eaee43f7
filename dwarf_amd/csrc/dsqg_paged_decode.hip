// Attention of one new token per sequence over a paged key/value cache (gfx950).
//
//   out[h] = sum_t w_t v_t,  w = softmax_t(scale q_h . k_t),  t = 0 .. pos
//
// One pass over the rows with a running maximum and sum: of the rows seen so far a group of lanes keeps
// m = max s_t, l = sum 2^(s_t - m) and acc = sum 2^(s_t - m) v_t (scores in base 2), and the parts of
// different rows join as  acc = sum_i 2^(m_i - m) acc_i.  Every key and value is read once and takes part
// in one product per query head, so memory bounds the step.
//
// A workgroup has one key/value head of one sequence, up to GT of the query heads that share it, and a
// chunk of the sequence's rows; its four waves take tiles in turn.  In a tile a row is 4, 8 or 16
// neighbouring lanes (RowMap), each wave load being whole rows of one page: a tile starts at a multiple of
// the wave's rows and a page is a multiple of them too, so the page number is the same for all lanes and
// comes from the table as a scalar.  Row groups keep statistics of their own until the chunk's end.
//
// Sequences longer than a chunk leave their chunks' (m, l, acc) in the workspace, and a second launch
// joins them in the order of the chunks.
//
// The first chunk's workgroup takes the new row from the caller's k_new and v_new (as the cache will hold
// it: through the 8-bit type's rounding), and stores it; no workgroup reads that row from the pool.
#include <algorithm>

#include "dsqg_launch.hpp"
#include "dsqg_mfma.hpp"
#include "dsqg_paged.hpp"

namespace dsqg {
namespace {

constexpr int kWaves = kBlock / 64;

// a + sum of the products of eight queries and eight key elements.
template <int QT, int CT>
__device__ __forceinline__ float dot8(const Raw8<QT>& qr, const float (&q)[8], const Raw8<CT>& kr, float a) {
  if constexpr (QT == DSQG_BF16 && CT == DSQG_BF16) {
    return dot8_bf16(qr.a, kr.a, a);
  } else {
    float k[8];
    raw_floats<CT>(kr, k);
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaf(q[i], k[i], a);
    return a;
  }
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
  constexpr int TR = U * R::rows;
  const int hg = (p.G + GT - 1) / GT;
  const int b = blockIdx.x / (p.c.Hkv * hg), rest = blockIdx.x - b * p.c.Hkv * hg;
  const int hk = rest / hg, g0 = (rest - hk * hg) * GT;
  const int split = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int gl = lane % R::lanes, r = lane / R::lanes;
  const int n = rows_of(p, b);
  const int chunks = chunks_of(p, n);
  if (split >= chunks) return;
  const long long h0 = (long long)b * p.H + hk * p.G + g0;  // first query head, in [B, H]
  if (n <= 0) {  // no rows: zeros; a position outside the table: NaN
    for (int e = threadIdx.x; e < GT * D; e += kBlock)
      if (g0 + e / D < p.G) store_out<QT>(p.out, h0 * D + e, n == 0 ? 0.f : __uint_as_float(0x7fc00000u));
    return;
  }

  const int* table = p.c.table + b * p.c.ts;
  const bool fresh = p.kn != nullptr;
  const int stored = stored_of(p, n);
  const int t0 = split * p.chunk, t1 = min(t0 + p.chunk, stored);

  Raw8<QT> qr[GT][PC];
  float q[GT][PC][8];
#pragma unroll
  for (int g = 0; g < GT; ++g)
#pragma unroll
    for (int u = 0; u < PC; ++u) {
      const int piece = gl + R::lanes * u;
      raw_zero<QT>(qr[g][u]);
      if (g0 + g < p.G && piece < R::CPR)
        qr[g][u] = raw_load<QT>(p.q + b * p.qb + (hk * p.G + g0 + g) * p.qh + piece * 8 * elem_size(QT));
      raw_floats<QT>(qr[g][u], q[g][u]);
    }

  Running<GT, PC> s;
  s.clear();

  if (fresh && split == 0 && wave == 0) {  // the new row, in the first row group
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
    const int t = n - 1, page = table[t >> p.c.shift];
    const bool ok = (unsigned)page < (unsigned)p.c.P;
    const float sk = narrow(CT) ? scale_value(kb) : 1.f, sv = narrow(CT) ? scale_value(vb) : 1.f;
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float d = 0.f;
#pragma unroll
      for (int u = 0; u < PC; ++u) d = dot8<QT, CT>(qr[g][u], q[g][u], kc[u], d);
      d = group_sum<R::lanes>(d) * (p.scale * sk);
      if (!ok) d = __uint_as_float(0x7fc00000u);  // nowhere to keep the row
      if (r == 0) {
        s.m[g] = fmaxf(d, -INFINITY);
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

  for (int tile = t0 + wave * TR; tile < t1; tile += kWaves * TR) {
    Raw8<CT> k[U][PC], v[U][PC];
    float sk[U], sv[U];
    bool bad[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (A pass that lies behind the last row reads that row's page, which exists, and is masked.)
      const int t = tile + u * R::rows;
      int page = table[min(t, stored - 1) >> p.c.shift];
      bad[u] = (unsigned)page >= (unsigned)p.c.P;
      page = bad[u] ? 0 : page;
      const long long slot = t & ((1 << p.c.shift) - 1);
      const char* kr = p.c.k + page * p.c.kp + hk * p.c.kh + slot * p.c.kn + r * p.c.kn;
      const char* vr = p.c.v + page * p.c.vp + hk * p.c.vh + slot * p.c.vn + r * p.c.vn;
#pragma unroll
      for (int w = 0; w < PC; ++w) {
        const int piece = gl + R::lanes * w;
        raw_zero<CT>(k[u][w]);
        raw_zero<CT>(v[u][w]);
        if (piece < R::CPR) {
          k[u][w] = raw_load<CT>(kr + piece * 8 * ES);
          v[u][w] = raw_load<CT>(vr + piece * 8 * ES);
        }
      }
      sk[u] = sv[u] = 1.f;
      if constexpr (narrow(CT)) {
        sk[u] = scale_value(p.c.ks[page * p.c.ksp + hk * p.c.ksh + (slot + r) * p.c.ksn]);
        sv[u] = scale_value(p.c.vs[page * p.c.vsp + hk * p.c.vsh + (slot + r) * p.c.vsn]);
      }
    }
    float sc[GT][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool live = tile + u * R::rows + r < t1;
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        float d = 0.f;
#pragma unroll
        for (int w = 0; w < PC; ++w) d = dot8<QT, CT>(qr[g][w], q[g][w], k[u][w], d);
        d = group_sum<R::lanes>(d) * (p.scale * sk[u]);
        if (bad[u]) d = __uint_as_float(0x7fc00000u);
        sc[g][u] = live ? d : -INFINITY;
      }
      // What lies behind the last row is no number of this sequence: zeros, so that 0 * value is 0.
      if (!live) {
        sv[u] = 0.f;
#pragma unroll
        for (int w = 0; w < PC; ++w) raw_zero<CT>(v[u][w]);
      }
    }
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float m = s.m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) m = fmaxf(m, sc[g][u]);
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
        sc[g][u] = e * sv[u];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int w = 0; w < PC; ++w) {
        float x[8];
        raw_floats<CT>(v[u][w], x);
#pragma unroll
        for (int g = 0; g < GT; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) s.acc[g][w][i] = fmaf(sc[g][u], x[i], s.acc[g][w][i]);
      }
  }

  // The row groups of the wave, then the waves through LDS.
  __shared__ float wm[kWaves][GT], wl[kWaves][GT], wacc[kWaves][GT][D];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    float m = s.m[g];
#pragma unroll
    for (int x = R::lanes; x < 64; x *= 2) m = fmaxf(m, __shfl_xor(m, x, 64));
    const float a = weight(s.m[g], m);
    float l = s.l[g] * a;
#pragma unroll
    for (int x = R::lanes; x < 64; x *= 2) l += __shfl_xor(l, x, 64);
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
        for (int y = R::lanes; y < 64; y *= 2) x += __shfl_xor(x, y, 64);
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
      const long long at = (h0 + g) * p.splits + split;
      p.acc[at * D + d] = x;
      if (d == 0) {
        p.ml[2 * at] = m;
        p.ml[2 * at + 1] = l;
      }
    }
  }
}

// Joins a head's chunks.  Grid: [B * H].  A chunk is JL lanes of four elements; the workgroup's rows of lanes
// take chunks in turn, each with a running maximum of its own, and meet in LDS: the order is fixed by the
// sequence's length alone.  Two memory round trips: the position, then every chunk's (m, l) and values.
template <int QT, int D>
__global__ __launch_bounds__(1024) void paged_join_kernel(PagedDecode p) {
  constexpr int JL = D <= 32 ? 8 : D <= 64 ? 16 : 32;
  const int b = blockIdx.x / p.H, rows = blockDim.x / JL;
  const int gl = threadIdx.x % JL, r = threadIdx.x / JL;
  const int chunks = chunks_of(p, rows_of(p, b));
  if (chunks == 1) return;  // (written by its only workgroup)
  const float2* ml = reinterpret_cast<const float2*>(p.ml) + (long long)blockIdx.x * p.splits;
  const float* acc = p.acc + (long long)blockIdx.x * p.splits * D + 4 * gl;
  constexpr int U = 4;
  float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = r; c0 < chunks; c0 += U * rows) {
    float2 s[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * rows;
      const bool live = c < chunks;
      s[u] = live ? ml[c] : make_float2(-INFINITY, 0.f);
      v[u] = live && 4 * gl < D ? *reinterpret_cast<const float4*>(acc + (long long)c * D) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) mn = fmaxf(mn, s[u].x);
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
  if (threadIdx.x >= D) return;
  const int n = min(rows, chunks);
  m = -INFINITY;
  for (int i = 0; i < n; ++i) m = fmaxf(m, jm[i]);
  float o = 0.f;
  l = 0.f;
  for (int i = 0; i < n; ++i) {
    const float w = weight(jm[i], m);
    l = fmaf(jl[i], w, l);
    o = fmaf(jx[i][threadIdx.x], w, o);
  }
  store_out<QT>(p.out, (long long)blockIdx.x * D + threadIdx.x, o / l);
}

// The kernels of a call and its split.
struct Plan {
  bool mfma;
  int heads;  // query heads of a workgroup
};

Plan plan(PagedDecode& p, int dtype, int cache_dtype, int D) {
  Plan k;
  k.mfma = p.G >= 2 && paged_mfma_takes(p, dtype, cache_dtype);
  // Three groups of eight a lane leave registers for two heads of the vector kernel.
  k.heads = k.mfma ? kMfmaHeads : p.G == 1 ? 1 : p.G == 2 || D == 80 || D == 96 ? 2 : 4;
  const long long T = std::max(1ll, (long long)p.c.M << p.c.shift);
  const long long units = (long long)p.c.B * p.c.Hkv * ((p.G + k.heads - 1) / k.heads);
  // Rows of a chunk: a few workgroups for each place on the chip, not so short that a workgroup's beginning
  // and end outweigh its rows.
  const long long most = k.mfma ? 1024 : 1536, least = k.mfma ? 256 : 128;
  long long chunk = ((T * units + most - 1) / most + 63) / 64 * 64;
  chunk = std::min(4096ll, std::max(least, chunk));
  chunk = std::max(chunk, (T / 65535 + 64) / 64 * 64);  // (the grid's limit)
  p.splits = (int)((T + chunk - 1) / chunk);
  p.chunk = (int)chunk;
  return k;
}

template <int QT, int CT, int D, int GT>
void launch(const PagedDecode& p, hipStream_t st) {
  const unsigned units = (unsigned)(p.c.B * p.c.Hkv * ((p.G + GT - 1) / GT));
  hipLaunchKernelGGL((paged_decode_kernel<QT, CT, D, GT>), dim3(units, (unsigned)p.splits), dim3(kBlock), 0, st, p);
}

template <int QT, int CT, int D>
void launch_heads(const PagedDecode& p, int heads, hipStream_t st) {
  if (heads == 1) {
    launch<QT, CT, D, 1>(p, st);
  } else if (heads == 2) {
    launch<QT, CT, D, 2>(p, st);
  } else if constexpr (RowMap<D>::pieces == 1) {
    launch<QT, CT, D, 4>(p, st);
  }
}

template <int QT, int D>
void launch_types(const PagedDecode& p, const Plan& k, int ct, hipStream_t st) {
  if (k.mfma) launch_paged_mfma(p, QT, ct, D, st);
  else if (ct == DSQG_E4M3) launch_heads<QT, DSQG_E4M3, D>(p, k.heads, st);
  else if (ct == DSQG_INT8) launch_heads<QT, DSQG_INT8, D>(p, k.heads, st);
  else launch_heads<QT, QT, D>(p, k.heads, st);
  if (p.splits > 1)
    hipLaunchKernelGGL((paged_join_kernel<QT, D>), dim3((unsigned)(p.c.B * p.H)), dim3(p.splits > 32 ? 1024 : 256), 0, st, p);
}

template <int QT>
void launch_dim(const PagedDecode& p, const Plan& k, int ct, int D, hipStream_t st) {
  switch (D) {
    case 32: launch_types<QT, 32>(p, k, ct, st); break;
    case 64: launch_types<QT, 64>(p, k, ct, st); break;
    case 80: launch_types<QT, 80>(p, k, ct, st); break;
    case 96: launch_types<QT, 96>(p, k, ct, st); break;
    default: launch_types<QT, 128>(p, k, ct, st); break;
  }
}

// The checks that the size query and the launch share; workspace bytes of the parts.
int check_decode(const dsqg_paged_decode_args* a, PagedDecode* p, Plan* k, size_t* bytes) {
  if (!a || a->H < 0) return DSQG_EINVAL;
  *p = PagedDecode{};
  *bytes = 0;
  if (const int st = check_paged_cache(a->cache, &p->c)) return st;
  const dsqg_paged_cache& c = a->cache;
  if (c.cache_dtype <= DSQG_F16 && c.cache_dtype != c.dtype) return DSQG_EINVAL;
  if (c.Hkv > 0 ? a->H % c.Hkv != 0 : a->H != 0) return DSQG_EINVAL;
  if ((long long)c.B * a->H == 0) return DSQG_OK;
  if ((long long)c.B * a->H >= (1ll << 23)) return DSQG_EUNSUPPORTED;  // grid: a workgroup of 256 a head
  p->H = a->H;
  p->G = a->H / c.Hkv;
  *k = plan(*p, c.dtype, c.cache_dtype, c.D);
  if (p->splits > 1) *bytes = (size_t)c.B * a->H * p->splits * (2 + c.D) * sizeof(float);
  return DSQG_OK;
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" int dsqg_paged_decode_workspace_size(const dsqg_paged_decode_args* a, size_t* bytes) {
  PagedDecode p;
  Plan k;
  return bytes ? check_decode(a, &p, &k, bytes) : (int)DSQG_EINVAL;
}

extern "C" int dsqg_paged_decode(const dsqg_paged_decode_args* a, dsqg_stream_t stream) {
  PagedDecode p;
  Plan k;
  size_t bytes = 0;
  if (const int st = check_decode(a, &p, &k, &bytes)) return st;
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
  if (bytes > 0) {
    if (!a->workspace || a->workspace_bytes < bytes) return DSQG_EWORKSPACE;
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return DSQG_EINVAL;
  }
  p.scale = a->softmax_scale * 1.4426950408889634f;
  p.q = static_cast<const char*>(a->q); p.qb = a->q_stride[0] * es; p.qh = a->q_stride[1] * es;
  p.kn = static_cast<const char*>(a->k_new); p.knb = a->k_new_stride[0] * es; p.knh = a->k_new_stride[1] * es;
  p.vn = static_cast<const char*>(a->v_new); p.vnb = a->v_new_stride[0] * es; p.vnh = a->v_new_stride[1] * es;
  p.pos = reinterpret_cast<const long long*>(a->pos);
  p.out = static_cast<char*>(a->out);
  p.acc = static_cast<float*>(a->workspace);
  p.ml = p.acc + (long long)c.B * a->H * p.splits * c.D;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (c.dtype == DSQG_F32) launch_dim<DSQG_F32>(p, k, c.cache_dtype, c.D, st);
  else if (c.dtype == DSQG_BF16) launch_dim<DSQG_BF16>(p, k, c.cache_dtype, c.D, st);
  else launch_dim<DSQG_F16>(p, k, c.cache_dtype, c.D, st);
  return hipGetLastError() == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
