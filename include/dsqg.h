/*
 * dsqg.h -- C ABI of libdsqg_hip.so, the MI355X (gfx950) DSQG fixed-offset sparse attention.
 *
 * DSQG attention: query row n of head (b,h) attends the J keys n - delta_j of the same head,
 * for a fixed, sorted offset table delta_0 < delta_1 < ... < delta_{J-1}.  With c = 1/sqrt(D):
 *
 *     s_j   = g[h,j] * c * q_n . k_{n-delta_j} + pos_bias[j,h] + c * q_n . se_j
 *     alpha = softmax_j(s) over the valid taps (n - delta_j >= 0); invalid taps have weight 0,
 *             are excluded from the normalisation and are never dereferenced
 *     out_n = a[h] * sum_j alpha_j v_{n-delta_j},     lse_n = logsumexp_j(s_j)
 *
 * g (score_gain, [H,J]) and a (if_gain, [H]) are optional (NULL means 1); se (scale_embed,
 * [J,D]) is optional (NULL means 0).  pos_bias is [J,H], as in the reference.
 *
 * Conventions.
 *  - Every entry point returns a dsqg_status.  Argument checks happen on the host before any
 *    HIP call, so a bad call never launches a kernel.
 *  - The library never allocates device memory and never synchronises; all work is ordered on
 *    the stream passed in.  Its only mutable global state is dsqg_bwd_noalloc's per-device
 *    static scratch (below); every other entry point is re-entrant.
 *  - Tensor pointers are device pointers.  Element strides are int64 element counts, in the
 *    order [B,H,N,D]; the innermost (D) stride must be 1 and the other strides and the base
 *    pointers must keep every row 16-byte aligned.
 *  - pos_bias / scale_embed / score_gain / if_gain and the parameter gradients are fp32 and
 *    contiguous; dsqg_fwd and dsqg_bwd also need scale_embed (when given) 16-byte aligned.  q/k/v/out/dout/dq/dk/dv share one element type (dtype).
 *
 * Reference interfaces replaced (paths are in the Lanerra/DWARF tree):
 *  - dsqg_fwd        <- _DSQGFnV3.forward, kernels/dsqg_attention_v3.py:361-387
 *                       (and the pybind forward(q,k,v,pb,se) of
 *                        kernels/dsqg_cuda/dsqg_cuda_kernel.cu:496-530)
 *  - dsqg_bwd        <- _DSQGFnV3.backward, kernels/dsqg_attention_v3.py:389-442
 *                       (pybind backward(...) of kernels/dsqg_cuda/dsqg_cuda_kernel.cu:532-609)
 *  - dsqg_decode_step: no counterpart in the reference, which regenerates the whole prefix for
 *                       every token (train/train_2048_condU.py:463-487); it realises the
 *                       circular K/V buffer described in README.md:175-177.
 *  - dsqg_pool_gate_fwd / _bwd <- the interference pool of DSQGBlock.forward,
 *                       train/train_2048_condU.py:289-292 (cumsum / counts, sigmoid gate), and
 *                       its autograd backward.
 */
#ifndef DWARF_DSQG_H
#define DWARF_DSQG_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DSQG_ABI_VERSION 9
#define DSQG_MAX_OFFSETS 64

/* Same type as hipStream_t; NULL is the null stream. */
typedef struct ihipStream_t* dsqg_stream_t;

typedef enum {
    DSQG_OK = 0,
    DSQG_EINVAL = 1,        /* bad shape, stride, alignment, pointer or offset table */
    DSQG_EUNSUPPORTED = 2,  /* valid arguments this build has no kernel for: the head dim,
                               J > 48, or (bf16) more than 16 offsets beyond the dense
                               window delta = 0, 1, 2, ... or a slice whose rows a 32-bit
                               byte offset cannot reach */
    DSQG_EHIP = 3,          /* a HIP launch failed (hipGetLastError after the launch) */
    DSQG_EWORKSPACE = 4,    /* workspace pointer NULL or smaller than required */
    DSQG_ETOOLARGE = 5      /* dsqg_bwd_noalloc: the call needs more than its static scratch */
} dsqg_status;

/* Static scratch of dsqg_bwd_noalloc (bytes per device): the backward workspace of the largest
 * call it takes, as dsqg_bwd_workspace_size reports it (e.g. 18 MB for bf16 B8 H12 N2048
 * D64 and the 44-offset table with dscale_embed, 10 MB without). */
#define DSQG_NOALLOC_SCRATCH_BYTES (64u << 20)

/* The attention over fixed offsets takes the first two; the entry points that say so take DSQG_F16, and
 * a paged cache also holds the 8-bit types (float8 e4m3 without infinities, and int8). */
typedef enum { DSQG_F32 = 0, DSQG_BF16 = 1, DSQG_F16 = 2, DSQG_E4M3 = 3, DSQG_INT8 = 4 } dsqg_dtype;

/* Shape and offset table shared by all entry points. */
typedef struct {
    int32_t dtype;                       /* dsqg_dtype */
    int32_t B, H, N, D;                  /* N is ignored by the decode step */
    int32_t J;                           /* number of offsets, 1..DSQG_MAX_OFFSETS; this
                                            build's kernels take J <= 48 (else EUNSUPPORTED) */
    int32_t offsets[DSQG_MAX_OFFSETS];   /* strictly increasing, offsets[0] == 0 */
} dsqg_shape;

/* Forward: out [B,H,N,D] (dtype), lse [B,H,N] fp32 contiguous (lse may be NULL).
 * alpha_lr (bf16 only; NULL = not written, and ignored for fp32): the softmax weights of the
 * long-range taps, [B,H,NS,N] fp32 contiguous with NS = dsqg_long_range_taps(offsets): saved
 * for the bf16 backward, which requires them (as the reference saves out and lse,
 * kernels/dsqg_attention_v3.py:384); dsqg_alpha_lr_elems gives its size.
 * Replaces kernels/dsqg_attention_v3.py:361-387 (_DSQGFnV3.forward). */
typedef struct {
    dsqg_shape shape;
    const void* q;  int64_t q_stride[4];
    const void* k;  int64_t k_stride[4];
    const void* v;  int64_t v_stride[4];
    const float* pos_bias;     /* [J,H] */
    const float* scale_embed;  /* [J,D] or NULL */
    const float* score_gain;   /* [H,J] or NULL */
    const float* if_gain;      /* [H]   or NULL */
    void* out;  int64_t out_stride[4];
    float* lse;                /* [B,H,N] or NULL */
    float* alpha_lr;           /* [B,H,NS,N] or NULL (bf16) */
} dsqg_fwd_args;

/* Backward.  dout is the gradient of out; lse and (bf16, required when the table has taps
 * beyond its dense window) alpha_lr are the forward's.  dq/dk/dv are written
 * (not accumulated).  dpos_bias [J,H] is required; dscale_embed [J,D], dscore_gain [H,J] and
 * dif_gain [H] are written when non-NULL (they are defined even when the matching input is
 * NULL, i.e. at se = 0, g = 1, a = 1).  The parameter gradients are reduced
 * deterministically from per-workgroup partials in the workspace (no global atomics).
 * Replaces kernels/dsqg_attention_v3.py:389-442 (_DSQGFnV3.backward). */
typedef struct {
    dsqg_shape shape;
    const void* q;    int64_t q_stride[4];
    const void* k;    int64_t k_stride[4];
    const void* v;    int64_t v_stride[4];
    const void* dout; int64_t dout_stride[4];
    const float* lse;          /* [B,H,N] */
    const float* pos_bias;     /* [J,H] */
    const float* scale_embed;  /* [J,D] or NULL */
    const float* score_gain;   /* [H,J] or NULL */
    const float* if_gain;      /* [H]   or NULL */
    void* dq;  int64_t dq_stride[4];
    void* dk;  int64_t dk_stride[4];
    void* dv;  int64_t dv_stride[4];
    float* dpos_bias;          /* [J,H] */
    float* dscale_embed;       /* [J,D] or NULL */
    float* dscore_gain;        /* [H,J] or NULL */
    float* dif_gain;           /* [H]   or NULL */
    void* workspace;           /* device memory, 256-byte aligned */
    size_t workspace_bytes;
    const float* alpha_lr;     /* [B,H,NS,N] from dsqg_fwd (bf16); ignored for fp32 */
} dsqg_bwd_args;

/* Decode step: one new token per sequence.  q, k_new, v_new, out are [B,H,D] contiguous;
 * k_ring, v_ring are [B,H,S,D] contiguous rings with S > max(offsets) and S*D*sizeof(dtype) < 2^31
 * (DSQG_EUNSUPPORTED otherwise).  pos [B] (device,
 * int64) is the absolute position of the new token.  The step writes k_new / v_new into slot
 * pos mod S, then attends slot (pos - delta_j) mod S for delta_j > 0 and the new row for
 * delta_j == 0; taps with pos - delta_j < 0 are masked (never wrapped).  If pos_next is non-NULL
 * (and distinct from pos) it receives pos + 1, so a captured step can be replayed.  A negative
 * pos marks an invalid sequence: its output is NaN, its rings are untouched, and pos_next
 * receives the same negative value, so it stays invalid over replays. */
typedef struct {
    dsqg_shape shape;
    int32_t S;                 /* ring slots */
    const void* q;
    const void* k_new;
    const void* v_new;
    void* k_ring;
    void* v_ring;
    const int64_t* pos;        /* [B] */
    int64_t* pos_next;         /* [B] or NULL */
    const float* pos_bias;     /* [J,H] */
    const float* scale_embed;  /* [J,D] or NULL */
    const float* score_gain;   /* [H,J] or NULL */
    const float* if_gain;      /* [H]   or NULL */
    void* out;
} dsqg_decode_args;

int dsqg_abi_version(void);
const char* dsqg_status_string(int status);

/* Head dims this build has kernels for, written to dims (up to cap entries); returns the
 * count. */
int dsqg_supported_head_dims(int32_t* dims, int cap);

int dsqg_fwd(const dsqg_fwd_args* args, dsqg_stream_t stream);

/* Taps beyond the dense window of an offset table (offsets[0..W] = 0..W, W <= 32): the NS of
 * alpha_lr.  Returns NS >= 0, or a negative DSQG_EINVAL for an invalid table. */
int dsqg_long_range_taps(const int32_t* offsets, int J);

/* Elements of alpha_lr for a shape (B * H * NS * N; 0 for fp32).  Returns DSQG_OK and writes
 * *elems, or an argument error.  No counterpart in the reference (which recomputes every score
 * in its backward). */
int dsqg_alpha_lr_elems(const dsqg_shape* shape, size_t* elems);

/* Workspace the backward needs for these arguments (shape and which gradients are requested).
 * Returns DSQG_OK and writes *bytes, or an argument error. */
int dsqg_bwd_workspace_size(const dsqg_bwd_args* args, size_t* bytes);
int dsqg_bwd(const dsqg_bwd_args* args, dsqg_stream_t stream);

/* The three phases dsqg_bwd runs, for callers that launch them separately (the reference's
 * backward is likewise three launches: kernels/dsqg_attention_v3.py:397-441).  Call them in
 * this order on one stream with the same args and workspace: the workspace carries D', (bf16)
 * the long-range taps' dk/dv weights and the parameter-gradient partials from phase 1 to
 * phases 2 and 3.
 *  - dsqg_bwd_dq     <- _compute_D_v3 + _bwd_dq_v3 (:397-424): dq, D', partials, and for bf16
 *                       the weights (c g dS, a alpha) of every query's long-range taps
 *  - dsqg_bwd_dkdv   <- _bwd_dkdv_v3 (:426-441): dk, dv
 *  - dsqg_bwd_params <- the tl.atomic_add accumulation of dpb/dse in _bwd_dq_v3 (:265-271),
 *                       here a deterministic reduction of the partials */
int dsqg_bwd_dq(const dsqg_bwd_args* args, dsqg_stream_t stream);
int dsqg_bwd_dkdv(const dsqg_bwd_args* args, dsqg_stream_t stream);
int dsqg_bwd_params(const dsqg_bwd_args* args, dsqg_stream_t stream);

/* dsqg_bwd without a workspace argument and without any allocation: no counterpart in the
 * reference.  For callers that cannot allocate device memory (code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc).  args->workspace and workspace_bytes
 * are ignored; the workspace is a static scratch array of DSQG_NOALLOC_SCRATCH_BYTES on each
 * device.  That array is part of the library's code object, so it takes its 64 MiB of device
 * memory on every device where the library is loaded, whether or not this entry point is ever
 * called.  Its address is looked up once per device on the first call there (hipGetSymbolAddress):
 * make that first call outside stream capture (one eager call), later calls may be captured
 * into a HIP graph (the call issues kernel launches only, no memset and no allocation).  A call whose
 * workspace (dsqg_bwd_workspace_size) exceeds it takes the launch plan with the smallest workspace
 * instead (dscale_embed partials over four batches each), and if that does not fit either returns
 * DSQG_ETOOLARGE before any HIP call.
 * Same kernels, outputs and stream rules as dsqg_bwd; calls that overlap on one device (other
 * streams, other threads) share the scratch and race, so serialise them. */
int dsqg_bwd_noalloc(const dsqg_bwd_args* args, dsqg_stream_t stream);

int dsqg_decode_step(const dsqg_decode_args* args, dsqg_stream_t stream);

/* K/V injection before the attention (train/train_2048_condU.py:178-181): with qkv [B,N,3*H*D] (unit
 * inner stride, element strides {b, n}) and deltas [B,H,N,D] (unit inner stride, strides {b, h, n}),
 * k_out = k + k_delta and v_out = v + v_delta, and q_out = q when given, each [B,N,H*D] with the
 * strides out_stride {b, n}; operands are rounded to out_dtype before the sum.  Types taken: all
 * F32, all BF16, or F16 in and BF16 out (EUNSUPPORTED otherwise).  D is a multiple of 8; bases and
 * strides keep every row 16-byte aligned. */
typedef struct {
    int32_t B, H, N, D;
    int32_t qkv_dtype, delta_dtype, out_dtype;
    const void* qkv;      int64_t qkv_stride[2];
    const void* k_delta;  int64_t k_delta_stride[3];
    const void* v_delta;  int64_t v_delta_stride[3];
    void* q_out;          /* or NULL */
    void* k_out;
    void* v_out;
    int64_t out_stride[2];
} dsqg_kv_inject_args;

int dsqg_kv_inject(const dsqg_kv_inject_args* args, dsqg_stream_t stream);

/* Loads a prompt into a layer's rings: row m of k and v [B,H,N,D], for m = max(0, N - S) .. N - 1,
 * goes to slot m mod S of k_ring and v_ring [B,H,S,D] (contiguous; other slots are untouched), and
 * pos [B] becomes N.  dtype F32, BF16 or F16, of all four; k and v have unit inner stride and the
 * other strides {b, h, n} and bases keep every row 16-byte aligned; D * sizeof(dtype) is a multiple
 * of 16 and B * H <= 65535 (EUNSUPPORTED otherwise).  No counterpart in the reference (README.md:
 * 175-179 describes the ring). */
typedef struct {
    int32_t dtype;
    int32_t B, H, N, S, D;
    const void* k;  int64_t k_stride[3];
    const void* v;  int64_t v_stride[3];
    void* k_ring;
    void* v_ring;
    int64_t* pos;
} dsqg_ring_load_args;

int dsqg_ring_load(const dsqg_ring_load_args* args, dsqg_stream_t stream);

/* Causal-mean pool with a sigmoid gate (the interference branch of a DWARF block):
 *
 *     pool[b,n,c] = (sum_{m<=n} x[b,m,c]) / (n + 1)
 *     out[b,n,c]  = s[b,n,c] * pool[b,n,c],         s = sigmoid(gate_pre), rounded to gate_dtype
 *
 * x, gate_pre and out are [B,N,C] with element strides {b, n} and unit channel stride; C must
 * be a multiple of 8, base pointers and rows 16-byte aligned, the row stride at least C (rows do
 * not overlap) and one batch slice under 2 GiB (EUNSUPPORTED otherwise).  Each tensor has its own element
 * type (F32, BF16 or F16); arithmetic is fp32 and the sums are deterministic.  The workspace
 * (size from dsqg_pool_gate_workspace_size, 256-byte aligned) holds per-chunk column sums.
 * Replaces train/train_2048_condU.py:289-292 (pool = xi.cumsum(1) / counts;
 * inter = sigmoid(inter_gate(xi)) * pool). */
typedef struct {
    int32_t B, N, C;
    int32_t x_dtype, gate_dtype, out_dtype;   /* dsqg_dtype each */
    const void* x;         int64_t x_stride[2];
    const void* gate_pre;  int64_t gate_stride[2];
    void* out;             int64_t out_stride[2];
    void* workspace;
    size_t workspace_bytes;
} dsqg_pool_gate_fwd_args;

/* Backward of dsqg_pool_gate_fwd for dout = d out (element type out_dtype):
 *
 *     dgate_pre[b,n,c] = dout * pool * s * (1 - s)                 (gate_dtype)
 *     dx[b,m,c]        = sum_{n>=m} dout[b,n,c] * s[b,n,c] / (n+1)  (x_dtype)
 *
 * Either output may be NULL (not computed).  Layout rules as for the forward.
 * Replaces torch autograd through train/train_2048_condU.py:289-292. */
typedef struct {
    int32_t B, N, C;
    int32_t x_dtype, gate_dtype, dout_dtype;  /* dsqg_dtype each */
    const void* x;         int64_t x_stride[2];
    const void* gate_pre;  int64_t gate_stride[2];
    const void* dout;      int64_t dout_stride[2];
    void* dx;              int64_t dx_stride[2];
    void* dgate_pre;       int64_t dgate_stride[2];
    void* workspace;
    size_t workspace_bytes;
} dsqg_pool_gate_bwd_args;

/* Workspace bytes of dsqg_pool_gate_fwd (backward == 0) or _bwd (backward != 0). */
int dsqg_pool_gate_workspace_size(int32_t B, int32_t N, int32_t C, int backward, size_t* bytes);
int dsqg_pool_gate_fwd(const dsqg_pool_gate_fwd_args* args, dsqg_stream_t stream);
int dsqg_pool_gate_bwd(const dsqg_pool_gate_bwd_args* args, dsqg_stream_t stream);

/* Weight and bias gradients of a linear layer y = x W^T + b (the layers around the attention,
 * train/train_2048_condU.py:126-130, 244-246): dw[o,i] = sum_t dy[t,o] x[t,i] and, when db is
 * given, db[o] = sum_t dy[t,o].  dy [T,O] and x [T,I] have unit column stride, row strides that are
 * a multiple of 8 elements and 16-byte aligned bases; O and I are multiples of 8, T >= 1; dw [O,I]
 * and db [O] are contiguous and 16-byte aligned.  Sums are fp32 and deterministic, rounded once to
 * out_dtype. */
typedef struct {
    int32_t T, O, I;
    int32_t dtype;             /* DSQG_F16 or DSQG_BF16, of dy and x */
    int32_t out_dtype;         /* that, or DSQG_F32, of dw and db */
    const void* dy;  int64_t dy_stride;
    const void* x;   int64_t x_stride;
    void* dw;
    void* db;                  /* or NULL */
    void* workspace;           /* 256-byte aligned */
    size_t workspace_bytes;
} dsqg_linear_wgrad_args;

int dsqg_linear_wgrad_workspace_size(const dsqg_linear_wgrad_args* args, size_t* bytes);
int dsqg_linear_wgrad(const dsqg_linear_wgrad_args* args, dsqg_stream_t stream);

/* A paged key/value cache of one layer (for full attention; train/train_2048_condU.py:210-245 keeps
 * none and recomputes the prefix).  k_pages and v_pages are pools [P, Hkv, page, D]; page_table [B, M]
 * says which page of the pools holds positions page * j .. page * (j + 1) - 1 of each sequence, so a
 * sequence has M * page positions at most.  Several sequences may share a page that none of them
 * writes.
 *
 * cache_dtype is dtype (that of the rows, queries and outputs) or an 8-bit type.  A row of an 8-bit
 * pool has a byte in k_scale / v_scale [P, Hkv, page]: value = code * 2^(byte - 127), with the smallest
 * power of two, 2^-127 at least, for which the row's largest magnitude is at most the type's largest
 * value (448 or 127); codes are rounded to nearest, ties to even.  A row that holds an infinity or NaN
 * gets byte 255 and reads as NaN.
 *
 * The kernels compare every page number with P and every position with M * page before they form an
 * address.  A row whose position has no page (a number below 0 or at least P, or a position past the
 * table) is not written; where it would be read, the result is NaN.
 *
 * page is a power of two from 16 to 65536, M * page at most 2^30; D is one of dsqg_supported_head_dims
 * (EUNSUPPORTED otherwise).  Pools have unit inner stride, other strides {page, head, row} in elements and
 * bases that keep every row 16-byte aligned, and rows that do not overlap; the scales' strides are
 * {page, head, row} as well.  B and Hkv are at most 65535.  (dsqg_paged_write and dsqg_paged_read: Hkv * N and
 * Hkv * T are less than 2^31.  dsqg_paged_decode: the page strides, and a page's rows times the row stride, are
 * less than 2^31 bytes, and B * H less than 2^21.) */
typedef struct {
    int32_t dtype;             /* DSQG_F32, DSQG_BF16 or DSQG_F16 */
    int32_t cache_dtype;       /* that, DSQG_E4M3 or DSQG_INT8 */
    int32_t B, Hkv, D;
    int32_t P, page, M;
    void* k_pages;     int64_t k_stride[3];
    void* v_pages;     int64_t v_stride[3];
    uint8_t* k_scale;  int64_t k_scale_stride[3];   /* NULL unless 8-bit */
    uint8_t* v_scale;  int64_t v_scale_stride[3];
    const int32_t* page_table;
    int64_t table_stride;      /* elements from one sequence's row to the next */
} dsqg_paged_cache;

/* Row i of sequence b of k and v [B,Hkv,N,D] (unit inner stride, strides {b, h, n}, rows 16-byte
 * aligned) goes to position pos[b] + i, for i < N and, where counts is given, i < counts[b]; every
 * other row of the pools stays as it is.  Where rows [B,N] is given (contiguous), row rows[b,i] of
 * k and v [B,Hkv,S,D], S = src_rows, goes there instead, and one whose number is none of theirs is not written. */
typedef struct {
    dsqg_paged_cache cache;
    int32_t N;
    const void* k;  int64_t k_stride[3];
    const void* v;  int64_t v_stride[3];
    const int64_t* pos;        /* [B] */
    const int64_t* counts;     /* [B] or NULL */
    const int64_t* rows;       /* [B,N] or NULL */
    int32_t src_rows;          /* with rows: rows of k and v */
} dsqg_paged_write_args;

int dsqg_paged_write(const dsqg_paged_write_args* args, dsqg_stream_t stream);

/* Positions t < lengths[b] of each sequence as k and v [B,Hkv,T,D] (contiguous, 16-byte aligned, of the
 * cache's dtype field, which here may differ from a 16- or 32-bit cache_dtype: values are rounded once);
 * rows t >= lengths[b] are zeros. */
typedef struct {
    dsqg_paged_cache cache;
    int32_t T;
    const int64_t* lengths;    /* [B] */
    void* k;
    void* v;
} dsqg_paged_read_args;

int dsqg_paged_read(const dsqg_paged_read_args* args, dsqg_stream_t stream);

/* Decode step: one new token per sequence.  q and out are [B,H,D], H a positive multiple of Hkv (query head h
 * attends key/value head h / (H / Hkv)), k_new and v_new [B,Hkv,D]; each but out (contiguous) has unit
 * inner stride, strides {b, h} and 16-byte aligned rows.  The step writes k_new and v_new to position
 * pos[b] (as dsqg_paged_write does) and gives
 *
 *     out[b,h] = sum_t softmax_t(softmax_scale * q . k_t) v_t      over t = 0 .. pos[b],
 *
 * of the rows as the cache holds them.  With k_new = v_new = NULL nothing is written and position pos[b]
 * is attended as it is.  A sequence with pos[b] < 0 attends nothing: its output is zeros and nothing is
 * written.  Sums and softmax statistics are fp32, in an order that does not change between calls.
 * Weights are kept relative to the largest, so the range is smaller than the types': values below 2^-90, and rows
 * of 8 bits whose largest is below 2^-70, lose bits or vanish; a row that weighs less than 2^-96 of the heaviest
 * (2^-140 in float16 pages) weighs nothing, and gives NaN where its value is infinite.  Queries over 8-bit pages
 * are below 2^112, so that their products with the codes are finite.
 * No two sequences may have the same page at the position that a step writes.
 * The workspace (256-byte aligned) holds the parts of sequences that are split over workgroups. */
typedef struct {
    dsqg_paged_cache cache;
    int32_t H;
    float softmax_scale;
    const void* q;      int64_t q_stride[2];
    const void* k_new;  int64_t k_new_stride[2];
    const void* v_new;  int64_t v_new_stride[2];
    const int64_t* pos;        /* [B] */
    void* out;
    void* workspace;
    size_t workspace_bytes;
} dsqg_paged_decode_args;

int dsqg_paged_decode_workspace_size(const dsqg_paged_decode_args* args, size_t* bytes);
int dsqg_paged_decode(const dsqg_paged_decode_args* args, dsqg_stream_t stream);

/* Softmax attention within a window, with sinks (the full-attention layer of train/train_2048_condU.py:210-245 sees all
 * earlier positions): position i of a sequence sees position j <= i if i - j < window or j < sinks.
 *
 *     out[b,h,i] = sum_j softmax_j(softmax_scale * q[b,h,i] . k[b,hk,j]) v[b,hk,j],    hk = h / (H / Hkv)
 *
 * q, out and their gradients are [B,H,N,D], k, v and theirs [B,Hkv,N,D], H a multiple of Hkv.  With lengths given, rows
 * i >= lengths[b] are not there: nothing sees them, and their outputs and gradients are zeros.  D is one of
 * dsqg_supported_head_dims (EUNSUPPORTED otherwise), window at least 1, sinks at least 0, N at most 2^30, and grids have less
 * than 2^32 lanes: B * H * ceil(N / 128) less than 2^24 and, in the backward, B * Hkv * (N / 64 + 33) less than 2^21 always do,
 * larger ones may not (EUNSUPPORTED).  Every tensor has unit inner stride, strides {b, h, n} and a base that keep rows
 * 16-byte aligned, and a row stride of at least D elements and less than 2^24 bytes.
 *
 * stats [B,H,N,2] (float, contiguous, 8-byte aligned; the forward's may be NULL) holds, for the backward, each query's
 * reference exponent and the inverse of its weights' sum, and low [B,H,N,D], of the inputs' 16-bit dtype, what out's rounding
 * took off (float16: times 2^11).  The backward takes dout . out from both; where low is NULL, from out alone, whose rounding
 * then shows in dq and dk: 3.5 times the error where a query sees few keys.  Scores and sums are fp32, in an order that does
 * not change between calls; the weights and, in the backward, their gradients are rounded once to a 16-bit dtype before they multiply
 * rows.  A row that a query does not see does not reach its output, whatever it holds, nor a row of a query that does not
 * see a key that key's gradients.
 *
 * Outputs are finite where the values are, up to 2^-7 below the type's largest.  Weights are kept relative to the largest: a row
 * that weighs less than 2^-96 of the heaviest (2^-38 in float16) weighs nothing, and gives an infinity or NaN where its value is
 * infinite. */
typedef struct {
    int32_t dtype;             /* DSQG_F32, DSQG_BF16 or DSQG_F16 */
    int32_t B, H, Hkv, N, D;
    int32_t window, sinks;
    float softmax_scale;
    const int64_t* lengths;    /* [B] or NULL */
} dsqg_window_shape;

typedef struct {
    dsqg_window_shape shape;
    const void* q;  int64_t q_stride[3];
    const void* k;  int64_t k_stride[3];
    const void* v;  int64_t v_stride[3];
    void* out;      int64_t out_stride[3];
    float* stats;
    void* low;      int64_t low_stride[3];     /* 16-bit dtypes, or NULL */
} dsqg_window_fwd_args;

int dsqg_window_fwd(const dsqg_window_fwd_args* args, dsqg_stream_t stream);

typedef struct {
    dsqg_window_shape shape;
    const void* q;     int64_t q_stride[3];
    const void* k;     int64_t k_stride[3];
    const void* v;     int64_t v_stride[3];
    const void* out;   int64_t out_stride[3];
    const void* dout;  int64_t dout_stride[3];
    const float* stats;
    const void* low;   int64_t low_stride[3];  /* 16-bit dtypes, or NULL */
    void* dq;  int64_t dq_stride[3];
    void* dk;  int64_t dk_stride[3];
    void* dv;  int64_t dv_stride[3];
    void* workspace;           /* 256-byte aligned */
    size_t workspace_bytes;
} dsqg_window_bwd_args;

int dsqg_window_bwd_workspace_size(const dsqg_window_shape* shape, size_t* bytes);
int dsqg_window_bwd(const dsqg_window_bwd_args* args, dsqg_stream_t stream);

/* The accepted path of a tree of drafted tokens (no counterpart in the reference).  Node i of sequence b has
 * the token tokens[b,i] and hangs on the node parents[b,i] (parents_stride 0: one tree for all); picks[b,i] is the
 * token that the model chose after node i.  Node 0 is accepted; from a node the walk goes to its first child behind it
 * whose token is the node's pick.  With counts given, only nodes i < counts[b] exist.
 *
 *     path[b,0..n[b]-1]: the nodes on the way, -1 behind them;  next[b]: the last one's pick
 *
 * A sequence without nodes has n = 0 and next = -1.  tokens and picks have unit inner stride, path [B,T], n [B] and
 * next [B] are contiguous; T is at most DSQG_MAX_TREE and B less than 2^26 (EUNSUPPORTED otherwise). */
#define DSQG_MAX_TREE 64

typedef struct {
    int32_t B, T;
    const int64_t* tokens;   int64_t tokens_stride;
    const int32_t* parents;  int64_t parents_stride;
    const int64_t* picks;    int64_t picks_stride;
    const int64_t* counts;     /* [B] or NULL */
    int64_t* path;
    int64_t* n;
    int64_t* next;
} dsqg_tree_accept_args;

int dsqg_tree_accept(const dsqg_tree_accept_args* args, dsqg_stream_t stream);

/* A step of T tokens of each sequence over a paged cache, drafted as a tree: k_new and v_new [B,Hkv,T,D] go to positions
 * pos[b] .. pos[b] + T - 1 (as dsqg_paged_write puts them there), and node i attends the positions before pos[b], its
 * ancestors and itself:
 *
 *     out[b,h,i] = sum_t softmax_t(softmax_scale * q[b,h,i] . k_t) v_t
 *
 * of the rows as the cache holds them (H a multiple of Hkv, as in dsqg_paged_decode).  Node i hangs on the earlier node
 * parents[b,i] or, -1, on the position before pos[b] (parents_stride 0: one tree for all; parents NULL: a chain).  With
 * counts given only nodes i < counts[b] exist.  What is no node, behind counts[b] or on parents that do not lead to -1
 * over earlier nodes, gets zeros; rows of the former are not written.
 *
 * With a window (0: none) a node at place pos[b] + depth sees the places above its own less window, and those below
 * sinks; a stored position is its own place.
 *
 * With k_new = v_new = NULL nothing is written and the draft's rows are attended as the pages hold them.  A sequence with
 * pos[b] < 0 is not in use: zeros, and nothing is written.  A node that sees a position without a page gets NaN.  A row
 * that a node does not see does not reach it, whatever it holds.  The range of values is dsqg_paged_decode's; its rules
 * for strides, q_stride {b, h, t} and so on, and workspace hold; out is contiguous [B,T,H,D].  Weights enter the sum as
 * two 16-bit terms where T * H / Hkv is at most 16, else as one (16-bit queries).  T is at most DSQG_MAX_TREE, B * H * T
 * less than 2^30, B * Hkv less than 2^24 - 8 and T * H / Hkv at most 2^21 - 32 (EUNSUPPORTED otherwise).  No two sequences
 * may have the same page at positions that a step writes. */
typedef struct {
    dsqg_paged_cache cache;
    int32_t H, T;
    int32_t window, sinks;
    float softmax_scale;
    const void* q;      int64_t q_stride[3];
    const void* k_new;  int64_t k_new_stride[3];
    const void* v_new;  int64_t v_new_stride[3];
    const int32_t* parents;  int64_t parents_stride;
    const int64_t* counts;     /* [B] or NULL */
    const int64_t* pos;        /* [B] */
    void* out;
    void* workspace;
    size_t workspace_bytes;
} dsqg_paged_tree_args;

int dsqg_paged_tree_workspace_size(const dsqg_paged_tree_args* args, size_t* bytes);
int dsqg_paged_tree(const dsqg_paged_tree_args* args, dsqg_stream_t stream);

/* A token of each row of logits by one number from [0, 1) (the reference's sampling, greedy or a nucleus,
 * train/train_2048_condU.py:474-484, with the limits in use since).  With w_i = exp((x_i - max x) / T) and the order of
 * x descending, of equal ones the lower index first, the tokens that stay are the first top_k, of those the ones
 * before which at most top_p of their mass lies, of those the ones with w >= min_p.
 *
 *     tokens[b] = the first i whose running mass, by index, is above u[b] times the mass that stays
 *     logprobs[b] = log(w / mass that stays)
 *
 * A temperature that is not above zero takes the largest logit (logprobs 0).  A NaN is no candidate, and neither is
 * -infinity; a row without candidates gives -1 and -infinity; infinities share a row's mass.  Masses are whole
 * multiples of 2^-F, F = 48 up to 2^14 tokens and 62 - ceil(log2 V) beyond, so that no result depends on an order.
 * top_k <= 0 or >= V, top_p >= 1 and min_p <= 0 limit nothing; min_p above 1 is 1.  A u that is not a
 * number or below 0 is 0, one of 1 or more takes the last token that stays.
 *
 * logits [B,V] have unit inner stride and any row stride and alignment (of an element); V is at most 2^30.  u is
 * float, or double where u_is_double.  A setting's array, where given, has the rows' own in the place of the
 * one for all, which must not be NaN. */
typedef struct {
    int32_t B, V;
    int32_t dtype;             /* DSQG_F32, DSQG_BF16 or DSQG_F16 */
    int32_t u_is_double;
    const void* logits;  int64_t logits_stride;
    const void* u;             /* [B] */
    double temperature, top_p, min_p;
    int64_t top_k;
    const float* temperatures; /* [B] or NULL, and so on */
    const int64_t* top_ks;
    const float* top_ps;
    const float* min_ps;
    int64_t* tokens;           /* [B] */
    float* logprobs;           /* [B] or NULL */
    void* workspace;           /* 256-byte aligned; may be NULL where its size is 0 */
    size_t workspace_bytes;
} dsqg_sample_args;

int dsqg_sample_workspace_size(int32_t B, int32_t V, int32_t dtype, size_t* bytes);
int dsqg_sample(const dsqg_sample_args* args, dsqg_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DWARF_DSQG_H */
