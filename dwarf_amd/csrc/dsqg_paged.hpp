// The paged key/value cache: launch parameters and element access shared by its kernels (gfx950).
//
// A pool of pages [P, Hkv, page, D] holds the keys of one layer, another one the values; a page is
// 2^shift consecutive positions of one sequence, and table[b][t >> shift] names the page of position
// t.  Every address that the kernels form starts from a page number that was compared with P first,
// and is 64 bits wide: a pool may be larger than 4 GiB.
//
// An 8-bit pool (e4m3 or int8) has one byte for each row of D values, the exponent of a power of two:
//   value = code * 2^(byte - 127),   byte 255: the row held an infinity or NaN and reads as NaN,
// with the smallest power of two (2^-127 at least) for which the row's largest magnitude is at most
// the type's largest value, 448 or 127.  A power of two makes the product with its inverse and the
// one on reading exact, so the code is the row's value rounded once (to nearest, ties to even), and
// what is read is the same in every kernel and in any order of operations.
#pragma once

#include "../../include/dsqg.h"
#include "dsqg_common.hpp"

namespace dsqg {

struct PagedCache {
  char* k; long long kp, kh, kn;             // strides in bytes: page, head, row
  char* v; long long vp, vh, vn;
  unsigned char* ks; long long ksp, ksh, ksn;
  unsigned char* vs; long long vsp, vsh, vsn;
  const int* table; long long ts;            // row stride in entries
  int B, Hkv, P, M, shift;
};

// DSQG_OK and the parameters, or an argument error; B * Hkv may be zero (nothing is checked then).
int check_paged_cache(const dsqg_paged_cache& a, PagedCache* c);

// ---- Elements in groups of eight. ------------------------------------------------------------------

typedef float f32x2v_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr bool narrow(int CT) { return CT == DSQG_E4M3 || CT == DSQG_INT8; }
constexpr int elem_size(int CT) { return CT == DSQG_F32 ? 4 : narrow(CT) ? 1 : 2; }

// Eight elements as they lie in memory.
template <int CT> struct Raw8 { uint4 a; };
template <> struct Raw8<DSQG_F32> { uint4 a, b; };
template <> struct Raw8<DSQG_E4M3> { uint2 a; };
template <> struct Raw8<DSQG_INT8> { uint2 a; };

template <int CT>
__device__ __forceinline__ Raw8<CT> raw_load(const void* p) { return *reinterpret_cast<const Raw8<CT>*>(p); }
template <int CT>
__device__ __forceinline__ void raw_store(void* p, const Raw8<CT>& x) { *reinterpret_cast<Raw8<CT>*>(p) = x; }

// The same past the caches' retention.
template <int CT>
__device__ __forceinline__ void raw_store_stream(void* p, const Raw8<CT>& x) {
  typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
  if constexpr (narrow(CT)) {
    __builtin_nontemporal_store(__builtin_bit_cast(u32x2_t, x.a), reinterpret_cast<u32x2_t*>(p));
  } else {
    st16_stream(p, x.a);
    if constexpr (CT == DSQG_F32) st16_stream(static_cast<char*>(p) + 16, x.b);
  }
}

template <int CT>
__device__ __forceinline__ void raw_zero(Raw8<CT>& x) { x = Raw8<CT>{}; }

template <int CT>
__device__ __forceinline__ void raw_floats(const Raw8<CT>& r, float (&x)[8]) {
  if constexpr (CT == DSQG_F32) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
  } else if constexpr (CT == DSQG_BF16) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else if constexpr (CT == DSQG_F16) {
    const f16x8_t h = __builtin_bit_cast(f16x8_t, r.a);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
  } else if constexpr (CT == DSQG_E4M3) {
    const uint32_t w[2] = {r.a.x, r.a.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2v_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
      const f32x2v_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
      x[4 * i] = lo[0]; x[4 * i + 1] = lo[1]; x[4 * i + 2] = hi[0]; x[4 * i + 3] = hi[1];
    }
  } else {
    const uint32_t w[2] = {r.a.x, r.a.y};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)(signed char)(w[i] >> (8 * j));
  }
}

// x rounded to nearest even into a 16- or 32-bit type (a value past float16's range becomes an infinity, as
// any conversion to that type makes it).
template <int CT>
__device__ __forceinline__ Raw8<CT> raw_round(const float (&x)[8]) {
  static_assert(!narrow(CT), "rows of 8 bits have scales");
  Raw8<CT> r;
  if constexpr (CT == DSQG_F32) {
    r.a = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    r.b = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
  } else if constexpr (CT == DSQG_BF16) {
    r.a = make_uint4(f32_to_bf16(x[0]) | (f32_to_bf16(x[1]) << 16), f32_to_bf16(x[2]) | (f32_to_bf16(x[3]) << 16),
                     f32_to_bf16(x[4]) | (f32_to_bf16(x[5]) << 16), f32_to_bf16(x[6]) | (f32_to_bf16(x[7]) << 16));
  } else {
    f16x8_t h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
    r.a = __builtin_bit_cast(uint4, h);
  }
  return r;
}

// The scale byte of a row whose largest magnitude is amax (NaN where the row holds one).
template <int CT>
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax) & 0x7fffffffu;
  if (u >= 0x7f800000u) return 255;
  // Largest values: 1.75 * 2^8 and 1.984375 * 2^6.  With amax = m * 2^x, m in [1, 2), the exponent is x less
  // 8 or 6, and one more where m is larger than that; a subnormal amax (u >> 23 = 0) ends at 2^-127.
  constexpr uint32_t top = CT == DSQG_E4M3 ? 0x600000u : 0x7e0000u;
  constexpr int x0 = CT == DSQG_E4M3 ? 8 : 6;
  const int e = (int)(u >> 23) - x0 + ((u & 0x7fffffu) > top ? 1 : 0);
  return e < 0 ? 0 : e;
}

// 2^(byte - 127); NaN for 255.
__device__ __forceinline__ float scale_value(int byte) {
  return __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : (uint32_t)byte << 23);
}

// Eight values of a row as codes under its scale byte (zeros under 255).
template <int CT>
__device__ __forceinline__ Raw8<CT> raw_encode(const float (&x)[8], int byte) {
  static_assert(narrow(CT), "8-bit types only");
  // 2^(127 - byte): 2^127 at byte 0, a normal number for every byte that scale_byte gives but 255.
  const float inv = byte == 255 ? 0.f : __uint_as_float((uint32_t)(254 - byte) << 23);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = byte == 255 ? 0.f : x[i] * inv;
  Raw8<CT> r;
  if constexpr (CT == DSQG_E4M3) {
    int a = 0, b = 0;
    a = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], a, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], a, true);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], b, false);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], b, true);
    r.a = make_uint2((uint32_t)a, (uint32_t)b);
  } else {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i / 4] |= ((uint32_t)(int)rintf(y[i]) & 0xffu) << (8 * (i % 4));
    r.a = make_uint2(w[0], w[1]);
  }
  return r;
}

// ---- Rows over lanes. ----------------------------------------------------------------------------------

// A row of D values is kRowLanes lanes (a power of two, so that sums run over aligned groups) of kRowPieces
// groups of eight each: lane l holds group l % kRowLanes + kRowLanes * u.  At D = 80 the last two of the
// twelve groups do not exist.
template <int D>
struct RowMap {
  static constexpr int CPR = D / 8;
  static constexpr int lanes = (CPR & (CPR - 1)) == 0 ? CPR : 4;
  static constexpr int pieces = (CPR + lanes - 1) / lanes;
  static constexpr int rows = 64 / lanes;  // rows of a wave's pass
};

// The larger of two magnitudes, as bits (no sign is set): a NaN is larger than an infinity and so is kept.
__device__ __forceinline__ float max_nan(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// Largest of x over aligned groups of G lanes (G = 4, 8, 16), in every lane.
template <int G>
__device__ __forceinline__ float group_max_nan(float x) {
  if constexpr (G >= 2) x = max_nan(x, dpp_f32<0xb1>(x));
  if constexpr (G >= 4) x = max_nan(x, dpp_f32<0x4e>(x));
  if constexpr (G >= 8) x = max_nan(x, dpp_f32<0x141>(x));
  if constexpr (G >= 16) x = max_nan(x, dpp_f32<0x140>(x));
  return x;
}

// A row of the caller's type DT as the pool keeps it.
template <int DT, int CT, int D>
__device__ __forceinline__ void put_row(char* dst, unsigned char* sc, const Raw8<DT> (&x)[RowMap<D>::pieces], int g) {
  using R = RowMap<D>;
  if constexpr (!narrow(CT)) {
    static_assert(DT == CT, "a 16- or 32-bit pool has the rows' type");
#pragma unroll
    for (int u = 0; u < R::pieces; ++u)
      if (g + R::lanes * u < R::CPR) raw_store<CT>(dst + (g + R::lanes * u) * 8 * elem_size(CT), x[u]);
  } else {
    float f[R::pieces][8], m = 0.f;
#pragma unroll
    for (int u = 0; u < R::pieces; ++u) {
      raw_floats<DT>(x[u], f[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(f[u][i]));
    }
    const int byte = scale_byte<CT>(group_max_nan<R::lanes>(m));
#pragma unroll
    for (int u = 0; u < R::pieces; ++u)
      if (g + R::lanes * u < R::CPR) raw_store<CT>(dst + (g + R::lanes * u) * 8, raw_encode<CT>(f[u], byte));
    if (g == 0) *sc = (unsigned char)byte;
  }
}

// ---- The decode step. -----------------------------------------------------------------------------------

// A step's work is split over workgroups in one of two ways.
//  * Chunks (shares = 0): a workgroup for each unit (a sequence's key/value head and up to `heads` of its query
//    heads) and chunk of `chunk` rows (all that the table holds, where it is short or units are many), as many
//    chunks as the longest sequence that the table could hold would have; those behind a sequence's end leave at
//    once.
//  * Shares: the rows of all units in one line, in steps of kShareRows, cut into `shares` equal parts, one a
//    workgroup: however the lengths differ, every workgroup has the same number of steps and no place on the chip
//    waits for the longest sequence.  A share may cover parts of several units; part w of unit u is number w + u
//    of the workspace, as one of the two grows from each part to the next.
// A unit that is not split is finished by its workgroup; the others' parts are joined by a second launch, for
// which the workgroup with a unit's first rows says how many there are, and where.
struct PagedDecode {
  PagedCache c;
  int H, G;            // query heads; of one key/value head
  float scale;         // softmax_scale * log2(e)
  const char* q; long long qb, qh;  // strides in bytes
  const char* kn; long long knb, knh;
  const char* vn; long long vnb, vnh;
  const long long* pos;
  char* out;           // [B, H, D]
  int heads;           // query heads of a unit, at most
  int chunk, splits;   // chunks: rows of one, a multiple of 64, and their number
  int shares;          // shares: their number
  int stream;          // rows are read past the caches' retention
  float* ml;           // workspace [parts, 2]: chunks [units, splits, heads], shares [shares + units, heads]
  float* acc;          // ... [parts, D]
  int2* joins;         // ... [units]: the first part, in `heads`, and how many
};

constexpr int kShareRows = 128;
constexpr int kShareSeqs = 512;  // sequences that a wave places its share among: eight a lane

// A load from memory that nothing writes while the kernel runs (positions, page numbers): of a uniform address a
// scalar load, which waits in no queue behind the rows' loads.
template <typename T>
__device__ __forceinline__ T load_const(const T* p) {
  typedef const __attribute__((address_space(4))) T* const_ptr;
  return *(const_ptr)(unsigned long long)p;
}

// Rows of sequence b that the step attends (0: none) or -1 where its position has no place in the table.
__device__ __forceinline__ int rows_at(const PagedDecode& p, long long pos) {
  if (pos < 0) return 0;
  return pos >= ((long long)p.c.M << p.c.shift) ? -1 : (int)pos + 1;
}

__device__ __forceinline__ int rows_of(const PagedDecode& p, int b) { return rows_at(p, load_const(p.pos + b)); }

// Rows that are read from the pool (the new one is not), and the chunks or steps that they make.
__device__ __forceinline__ int stored_of(const PagedDecode& p, int n) { return p.kn ? n - 1 : n; }
__device__ __forceinline__ int chunks_of(const PagedDecode& p, int n) {
  return n <= 0 ? 1 : max(1, (stored_of(p, n) + p.chunk - 1) / p.chunk);
}
__device__ __forceinline__ int steps_of(const PagedDecode& p, int n) {
  return n <= 0 ? 1 : max(1, (stored_of(p, n) + kShareRows - 1) / kShareRows);
}

// Where the units lie in the line of steps: a wave's view, for up to kShareSeqs sequences, whose rows it holds
// eight a lane.
struct ShareLine {
  int n[kShareSeqs / 64], sum, incl, q;  // this lane's sequences' rows, their steps, and the steps up to them
  int units, per;                        // units of a sequence; steps of a share
  __device__ __forceinline__ ShareLine(const PagedDecode& p) {
    const int l = threadIdx.x & 63;
    q = (p.c.B + 63) / 64;
    units = p.c.Hkv * ((p.G + p.heads - 1) / p.heads);
#pragma unroll
    for (int j = 0; j < kShareSeqs / 64; ++j) n[j] = j < q && l * q + j < p.c.B ? rows_of(p, l * q + j) : 0;
    sum = 0;
#pragma unroll
    for (int j = 0; j < kShareSeqs / 64; ++j) sum += j < q && l * q + j < p.c.B ? steps_of(p, n[j]) : 0;
    // Inclusive sums over the lanes: inside rows of 16, then rows 0 and 2 into 1 and 3, then the first half
    // into the second.
    incl = sum;
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x111, 0xf, 0xf, true);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x112, 0xf, 0xf, true);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x114, 0xf, 0xf, true);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x118, 0xf, 0xf, true);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x142, 0xa, 0xf, false);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x143, 0xc, 0xf, false);
    const int total = steps();
    per = (total + p.shares - 1) / p.shares;
  }
  __device__ __forceinline__ int steps() const { return __builtin_amdgcn_readlane(incl, 63) * units; }
  // Rows of sequence b, and the line's steps before it.
  __device__ __forceinline__ int rows(int b) const {
    const int lane = b / q, j0 = b - lane * q;
    int r = 0;
#pragma unroll
    for (int j = 0; j < kShareSeqs / 64; ++j)
      if (j == j0) r = __builtin_amdgcn_readlane(n[j], lane);
    return r;
  }
  __device__ __forceinline__ int before(const PagedDecode& p, int b) const {
    const int lane = b / q, j0 = b - lane * q;
    int r = __builtin_amdgcn_readlane(incl, lane) - __builtin_amdgcn_readlane(sum, lane);
#pragma unroll
    for (int j = 0; j < kShareSeqs / 64; ++j)
      if (j < j0) r += steps_of(p, __builtin_amdgcn_readlane(n[j], lane));
    return r * units;
  }
  // The sequence that step s belongs to (s < steps()).
  __device__ __forceinline__ int sequence(const PagedDecode& p, int s) const {
    const int lane = __builtin_ctzll(__ballot(s < incl * units));
    int at = (__builtin_amdgcn_readlane(incl, lane) - __builtin_amdgcn_readlane(sum, lane)) * units, b = lane * q;
#pragma unroll
    for (int j = 0; j < kShareSeqs / 64 - 1; ++j)
      if (j < q - 1) {
        const int next = at + steps_of(p, __builtin_amdgcn_readlane(n[j], lane)) * units;
        if (s >= next && b == lane * q + j) {
          at = next;
          ++b;
        }
      }
    return b;
  }
};

template <int QT>
__device__ __forceinline__ void store_out(char* out, long long e, float x) {
  if constexpr (QT == DSQG_F32) reinterpret_cast<float*>(out)[e] = x;
  else if constexpr (QT == DSQG_BF16) reinterpret_cast<bf16_t*>(out)[e] = (bf16_t)f32_to_bf16(x);
  else reinterpret_cast<_Float16*>(out)[e] = (_Float16)x;
}

// 2^(a - b), where b is the larger: 0 for a = -inf also where b is, NaN for a NaN (which the maxima that
// b comes from pass over, so that the sums carry it).  a is a score as its maximum was taken of it, rounded: the
// exact product in one multiply-add with b would leave that rounding as an exponent, past 2^26 one without bounds.
__device__ __forceinline__ float weight(float a, float b) {
#pragma clang fp contract(off)
  return __builtin_amdgcn_exp2f(a - (b == -INFINITY ? 0.f : b));
}

// The largest weight is 2^lift, not 1: sums of 2^30 rows of the largest float32 or bfloat16 value stay finite, as
// their mean is, until the last division (and values above 2^-96 keep their precision); in float16 products
// weights are larger instead, so that small ones stay clear of its subnormal numbers.
template <bool F16>
constexpr float weight_lift() { return F16 ? 14.f : -30.f; }

// What a row of the largest score m is weighed against (no multiply-add either).
template <bool F16>
__device__ __forceinline__ float lifted(float m) {
#pragma clang fp contract(off)
  return m - weight_lift<F16>();
}

// Largest group of query heads that one workgroup of the matrix-instruction kernel takes.
constexpr int kMfmaHeads = 16;

// The matrix-instruction kernel (dsqg_paged_mfma.hip): whether it takes these types and layouts, and its launch
// over p.splits chunks (the join is the caller's).
bool paged_mfma_takes(const PagedDecode& p, int dtype, int cache_dtype);
void launch_paged_mfma(const PagedDecode& p, int dtype, int cache_dtype, int D, hipStream_t st);
// Workgroups of it that the chip holds, and whether it takes shares of these rows.
int paged_mfma_places(int D);
constexpr bool paged_mfma_shares(int cache_dtype, int D) { return D < 128 || narrow(cache_dtype); }

}  // namespace dsqg
