// Writing rows into a paged key/value cache and reading them back (gfx950); the cache's layout and the
// 8-bit types' scales are described in dsqg_paged.hpp.
//
// Both move every value once and compute next to nothing, so memory bounds them: a lane takes eight
// elements of a key row and the same eight of the value row, a row being 4, 8 or 16 neighbouring lanes
// (four lanes of three groups at D = 80 and 96), so that a wave's accesses are whole rows.  The largest
// magnitude that a scale needs is a maximum over those lanes (DPP), without LDS or a second pass.
// Medians: 8 x 2048 positions, 12 heads of 64, from bfloat16 into e4m3 (76 MB): 15.8 us, 4.8 TB/s, a copy's rate;
// 16 x 4096 positions (63 % of them in use), 8 heads of 128, from int8 to float16 (354 MB): 60 us, 5.9 TB/s;
// 2 x 65536, 8 heads of 128, from e4m3 to bfloat16 (807 MB): 162 us, 5.0 TB/s (147 at the least).
#include <algorithm>

#include "dsqg_launch.hpp"
#include "dsqg_mfma.hpp"
#include "dsqg_paged.hpp"

namespace dsqg {

int check_paged_cache(const dsqg_paged_cache& a, PagedCache* c) {
  const bool small = a.cache_dtype == DSQG_E4M3 || a.cache_dtype == DSQG_INT8;
  if (a.dtype < DSQG_F32 || a.dtype > DSQG_F16) return DSQG_EINVAL;
  if (a.cache_dtype < DSQG_F32 || a.cache_dtype > DSQG_INT8) return DSQG_EINVAL;
  if (a.B < 0 || a.Hkv < 0 || a.D <= 0 || a.P < 0 || a.M < 0 || a.page <= 0) return DSQG_EINVAL;
  if ((a.page & (a.page - 1)) != 0) return DSQG_EINVAL;
  if (!head_dim_supported(a.D) || a.page < 16 || a.page > 65536) return DSQG_EUNSUPPORTED;
  if ((long long)a.M * a.page > (1ll << 30) || a.B > 65535 || a.Hkv > 65535) return DSQG_EUNSUPPORTED;
  *c = PagedCache{};
  c->B = a.B; c->Hkv = a.Hkv; c->P = a.P; c->M = a.M;
  while ((1 << c->shift) < a.page) ++c->shift;
  if ((long long)a.B * a.Hkv == 0) return DSQG_OK;
  if (a.P == 0) return DSQG_EINVAL;  // a pool without pages holds nothing
  const long long es = elem_size(a.cache_dtype);
  // A pool: a base, three strides (bytes) and the bytes of a row; rows must not overlap.
  auto pool = [&](const void* base, const int64_t st[3], long long e, long long row, long long align) {
    if (!base || (reinterpret_cast<uintptr_t>(base) & (align - 1)) != 0) return false;
    long long s[3], n[3] = {a.P, a.Hkv, a.page};
    for (int i = 0; i < 3; ++i) {
      if (st[i] < 0 || st[i] > (1ll << 50) || (st[i] * e) % align != 0) return false;
      s[i] = st[i] * e;
    }
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < 2 - i; ++j)
        if (s[j] > s[j + 1]) {
          long long x = s[j]; s[j] = s[j + 1]; s[j + 1] = x;
          x = n[j]; n[j] = n[j + 1]; n[j + 1] = x;
        }
    long long extent = row;
    for (int i = 0; i < 3; ++i) {
      if (n[i] > 1 && s[i] < extent) return false;
      extent += (n[i] - 1) * s[i];
    }
    return true;
  };
  if (!pool(a.k_pages, a.k_stride, es, a.D * es, 16) || !pool(a.v_pages, a.v_stride, es, a.D * es, 16)) return DSQG_EINVAL;
  if (small && (!pool(a.k_scale, a.k_scale_stride, 1, 1, 1) || !pool(a.v_scale, a.v_scale_stride, 1, 1, 1)))
    return DSQG_EINVAL;
  if (a.M > 0 && (!a.page_table || a.table_stride < 0 || a.table_stride > (1ll << 50))) return DSQG_EINVAL;
  c->k = static_cast<char*>(a.k_pages);
  c->kp = a.k_stride[0] * es; c->kh = a.k_stride[1] * es; c->kn = a.k_stride[2] * es;
  c->v = static_cast<char*>(a.v_pages);
  c->vp = a.v_stride[0] * es; c->vh = a.v_stride[1] * es; c->vn = a.v_stride[2] * es;
  if (small) {
    c->ks = a.k_scale; c->ksp = a.k_scale_stride[0]; c->ksh = a.k_scale_stride[1]; c->ksn = a.k_scale_stride[2];
    c->vs = a.v_scale; c->vsp = a.v_scale_stride[0]; c->vsh = a.v_scale_stride[1]; c->vsn = a.v_scale_stride[2];
  }
  c->table = a.page_table; c->ts = a.table_stride;
  return DSQG_OK;
}

namespace {

// Rows of one sequence that a grid takes (sixteen lanes a row, below 2^32 lanes in x); more are several launches,
// up to a limit that outputs cannot reach (2^31 rows are 274 GB at least).
constexpr long long kGridRows = 1ll << 27, kMostRows = 1ll << 31;

struct WriteParams {
  PagedCache c;
  const char* k; long long kb, kh, kn;  // strides in bytes
  const char* v; long long vb, vh, vn;
  const long long* pos; const long long* counts;
  const long long* src;  // [B, N]: rows of k and v, below S, in the place of 0 .. N - 1; or null
  int N, S;
  long long rows;  // Hkv * N of one sequence
  long long row0;  // the launch's first
};

struct ReadParams {
  PagedCache c;
  const long long* lengths;
  char* k; char* v;
  int T;
  bool stream;     // the output is larger than the caches that the next launch could find it in
  long long rows;  // Hkv * T of one sequence
  long long row0;  // the launch's first
};

// Grid: x over rows (h, n) of a sequence, n fastest; y over sequences.
template <int DT, int CT, int D>
__global__ __launch_bounds__(kBlock) void paged_write_kernel(WriteParams p) {
  using R = RowMap<D>;
  constexpr int rpb = kBlock / R::lanes;
  const int b = blockIdx.y, g = threadIdx.x % R::lanes;
  const long long row = p.row0 + (long long)blockIdx.x * rpb + threadIdx.x / R::lanes;
  if (row >= p.rows) return;
  const int h = (int)(row / p.N), n = (int)(row - (long long)h * p.N);
  if (p.counts && n >= p.counts[b]) return;
  const long long t = p.pos[b] + n;
  if (t < 0 || t >= ((long long)p.c.M << p.c.shift)) return;
  const int page = p.c.table[b * p.c.ts + (t >> p.c.shift)];
  if ((unsigned)page >= (unsigned)p.c.P) return;
  const long long from = p.src ? p.src[(long long)b * p.N + n] : n;
  if ((unsigned long long)from >= (unsigned long long)p.S) return;
  const long long slot = t & ((1 << p.c.shift) - 1);
  const char* ks = p.k + b * p.kb + h * p.kh + from * p.kn;
  const char* vs = p.v + b * p.vb + h * p.vh + from * p.vn;
  Raw8<DT> x[R::pieces], y[R::pieces];
#pragma unroll
  for (int u = 0; u < R::pieces; ++u) {
    raw_zero<DT>(x[u]);
    raw_zero<DT>(y[u]);
    if (g + R::lanes * u < R::CPR) {
      x[u] = raw_load<DT>(ks + (g + R::lanes * u) * 8 * elem_size(DT));
      y[u] = raw_load<DT>(vs + (g + R::lanes * u) * 8 * elem_size(DT));
    }
  }
  put_row<DT, CT, D>(p.c.k + page * p.c.kp + h * p.c.kh + slot * p.c.kn,
                     p.c.ks + page * p.c.ksp + h * p.c.ksh + slot * p.c.ksn, x, g);
  put_row<DT, CT, D>(p.c.v + page * p.c.vp + h * p.c.vh + slot * p.c.vn,
                     p.c.vs + page * p.c.vsp + h * p.c.vsh + slot * p.c.vsn, y, g);
}

// Eight elements of a stored row in the output's type.
template <int CT, int OT>
__device__ __forceinline__ Raw8<OT> get_piece(const Raw8<CT>& r, float scale) {
  if constexpr (CT == OT) {
    return r;
  } else {
    float x[8];
    raw_floats<CT>(r, x);
    if constexpr (narrow(CT)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= scale;
    }
    return raw_round<OT>(x);
  }
}

// Grid: as the write's, over the T positions of the output.  (STREAM: a parameter, as two stores in two branches
// become one that is neither.)
template <int CT, int OT, int D, bool STREAM>
__global__ __launch_bounds__(kBlock) void paged_read_kernel(ReadParams p) {
  using R = RowMap<D>;
  constexpr int rpb = kBlock / R::lanes;
  const int b = blockIdx.y, g = threadIdx.x % R::lanes;
  const long long row = p.row0 + (long long)blockIdx.x * rpb + threadIdx.x / R::lanes;
  if (row >= p.rows) return;
  const int h = (int)(row / p.T), t = (int)(row - (long long)h * p.T);
  const long long out = ((long long)b * p.rows + row) * D * elem_size(OT);
  const bool live = t < p.lengths[b];
  int page = -1;
  if (live && (t >> p.c.shift) < p.c.M) page = p.c.table[b * p.c.ts + (t >> p.c.shift)];
  Raw8<OT> x[R::pieces], y[R::pieces];
  if ((unsigned)page < (unsigned)p.c.P) {
    const int slot = t & ((1 << p.c.shift) - 1);
    const char* ks = p.c.k + page * p.c.kp + h * p.c.kh + slot * p.c.kn;
    const char* vs = p.c.v + page * p.c.vp + h * p.c.vh + slot * p.c.vn;
    float sk = 1.f, sv = 1.f;
    if constexpr (narrow(CT)) {
      sk = scale_value(p.c.ks[page * p.c.ksp + h * p.c.ksh + slot * p.c.ksn]);
      sv = scale_value(p.c.vs[page * p.c.vsp + h * p.c.vsh + slot * p.c.vsn]);
    }
#pragma unroll
    for (int u = 0; u < R::pieces; ++u)
      if (g + R::lanes * u < R::CPR) {
        x[u] = get_piece<CT, OT>(raw_load<CT>(ks + (g + R::lanes * u) * 8 * elem_size(CT)), sk);
        y[u] = get_piece<CT, OT>(raw_load<CT>(vs + (g + R::lanes * u) * 8 * elem_size(CT)), sv);
      }
  } else {
    // Behind the sequence's end: zeros.  A position without a page: NaN.
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = live ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
    for (int u = 0; u < R::pieces; ++u) x[u] = y[u] = raw_round<OT>(f);
  }
#pragma unroll
  for (int u = 0; u < R::pieces; ++u)
    if (g + R::lanes * u < R::CPR) {
      const long long at = out + (g + R::lanes * u) * 8 * elem_size(OT);
      if constexpr (STREAM) {
        raw_store_stream<OT>(p.k + at, x[u]);
        raw_store_stream<OT>(p.v + at, y[u]);
      } else {
        raw_store<OT>(p.k + at, x[u]);
        raw_store<OT>(p.v + at, y[u]);
      }
    }
}

// The rows in launches of what a grid takes: f(its grid), p.row0 being its first row.
template <int D, typename P, typename F>
void for_grids(P p, F&& f) {
  constexpr int rpb = kBlock / RowMap<D>::lanes;
  for (; p.row0 < p.rows; p.row0 += kGridRows) {
    const long long n = std::min(p.rows - p.row0, kGridRows);
    f(p, dim3((unsigned)((n + rpb - 1) / rpb), (unsigned)p.c.B));
  }
}

template <int DT, int CT, int D>
void launch_write(const WriteParams& a, hipStream_t st) {
  for_grids<D>(a, [&](const WriteParams& p, dim3 grid) {
    hipLaunchKernelGGL((paged_write_kernel<DT, CT, D>), grid, dim3(kBlock), 0, st, p);
  });
}

template <int CT, int OT, int D>
void launch_read(const ReadParams& a, hipStream_t st) {
  for_grids<D>(a, [&](const ReadParams& p, dim3 grid) {
    if (p.stream) hipLaunchKernelGGL((paged_read_kernel<CT, OT, D, true>), grid, dim3(kBlock), 0, st, p);
    else hipLaunchKernelGGL((paged_read_kernel<CT, OT, D, false>), grid, dim3(kBlock), 0, st, p);
  });
}

template <int DT, int D>
void write_dtype(const WriteParams& p, int ct, hipStream_t st) {
  if (ct == DSQG_E4M3) launch_write<DT, DSQG_E4M3, D>(p, st);
  else if (ct == DSQG_INT8) launch_write<DT, DSQG_INT8, D>(p, st);
  else launch_write<DT, DT, D>(p, st);
}

template <int OT, int D>
void read_dtype(const ReadParams& p, int ct, hipStream_t st) {
  switch (ct) {
    case DSQG_F32: launch_read<DSQG_F32, OT, D>(p, st); break;
    case DSQG_BF16: launch_read<DSQG_BF16, OT, D>(p, st); break;
    case DSQG_F16: launch_read<DSQG_F16, OT, D>(p, st); break;
    case DSQG_E4M3: launch_read<DSQG_E4M3, OT, D>(p, st); break;
    default: launch_read<DSQG_INT8, OT, D>(p, st); break;
  }
}

// Calls F<D>::run for a head dim that head_dim_supported takes.
template <template <int> class F, typename... A>
void for_dim(int D, A&&... a) {
  switch (D) {
    case 32: F<32>::run(a...); break;
    case 64: F<64>::run(a...); break;
    case 80: F<80>::run(a...); break;
    case 96: F<96>::run(a...); break;
    default: F<128>::run(a...); break;
  }
}

template <int D>
struct WriteDim {
  static void run(const WriteParams& p, int dt, int ct, hipStream_t st) {
    if (dt == DSQG_F32) write_dtype<DSQG_F32, D>(p, ct, st);
    else if (dt == DSQG_BF16) write_dtype<DSQG_BF16, D>(p, ct, st);
    else write_dtype<DSQG_F16, D>(p, ct, st);
  }
};

template <int D>
struct ReadDim {
  static void run(const ReadParams& p, int ot, int ct, hipStream_t st) {
    if (ot == DSQG_F32) read_dtype<DSQG_F32, D>(p, ct, st);
    else if (ot == DSQG_BF16) read_dtype<DSQG_BF16, D>(p, ct, st);
    else read_dtype<DSQG_F16, D>(p, ct, st);
  }
};

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" int dsqg_paged_write(const dsqg_paged_write_args* a, dsqg_stream_t stream) {
  if (!a || a->N < 0) return DSQG_EINVAL;
  WriteParams p = {};
  if (const int st = check_paged_cache(a->cache, &p.c)) return st;
  const dsqg_paged_cache& c = a->cache;
  if (c.cache_dtype <= DSQG_F16 && c.cache_dtype != c.dtype) return DSQG_EINVAL;
  if ((long long)c.B * c.Hkv * a->N == 0) return DSQG_OK;
  const long long es = elem_size(c.dtype);
  auto bad = [](const void* ptr) { return !ptr || (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0; };
  const bool none = a->rows && a->src_rows == 0;  // (nothing to take rows from: no pointers either)
  if ((!none && (bad(a->k) || bad(a->v))) || !a->pos) return DSQG_EINVAL;
  for (int i = 0; i < 3; ++i)
    if (a->k_stride[i] < 0 || a->v_stride[i] < 0 || a->k_stride[i] > (1ll << 50) || a->v_stride[i] > (1ll << 50) ||
        a->k_stride[i] * es % 16 != 0 || a->v_stride[i] * es % 16 != 0)
      return DSQG_EINVAL;
  p.k = static_cast<const char*>(a->k); p.kb = a->k_stride[0] * es; p.kh = a->k_stride[1] * es; p.kn = a->k_stride[2] * es;
  p.v = static_cast<const char*>(a->v); p.vb = a->v_stride[0] * es; p.vh = a->v_stride[1] * es; p.vn = a->v_stride[2] * es;
  p.pos = reinterpret_cast<const long long*>(a->pos);
  p.counts = reinterpret_cast<const long long*>(a->counts);
  p.src = reinterpret_cast<const long long*>(a->rows);
  if (p.src && a->src_rows < 0) return DSQG_EINVAL;
  p.N = a->N;
  p.S = p.src ? a->src_rows : a->N;
  if (p.S == 0) return DSQG_OK;
  p.rows = (long long)c.Hkv * a->N;
  if (p.rows >= kMostRows) return DSQG_EUNSUPPORTED;
  for_dim<WriteDim>(c.D, p, c.dtype, c.cache_dtype, reinterpret_cast<hipStream_t>(stream));
  return hipGetLastError() == hipSuccess ? DSQG_OK : DSQG_EHIP;
}

extern "C" int dsqg_paged_read(const dsqg_paged_read_args* a, dsqg_stream_t stream) {
  if (!a || a->T < 0) return DSQG_EINVAL;
  ReadParams p = {};
  if (const int st = check_paged_cache(a->cache, &p.c)) return st;
  const dsqg_paged_cache& c = a->cache;
  if ((long long)c.B * c.Hkv * a->T == 0) return DSQG_OK;
  auto bad = [](const void* ptr) { return !ptr || (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0; };
  if (bad(a->k) || bad(a->v) || !a->lengths) return DSQG_EINVAL;
  p.lengths = reinterpret_cast<const long long*>(a->lengths);
  p.k = static_cast<char*>(a->k);
  p.v = static_cast<char*>(a->v);
  p.T = a->T;
  p.rows = (long long)c.Hkv * a->T;
  if (p.rows >= kMostRows) return DSQG_EUNSUPPORTED;
  // Results that the eight L2s (32 MB) cannot hold push the pool's lines out of them for nothing: 537 MB of them
  // leave in 161 to 163 us, 168 to 170 the ordinary way (medians of two runs each).  Smaller ones are left where
  // the next launch finds them.
  p.stream = 2ll * c.B * p.rows * c.D * elem_size(c.dtype) > (32ll << 20);
  for_dim<ReadDim>(c.D, p, c.dtype, c.cache_dtype, reinterpret_cast<hipStream_t>(stream));
  return hipGetLastError() == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
