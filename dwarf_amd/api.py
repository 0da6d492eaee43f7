"""Public DSQG entry points with the reference's signatures and dtype rules.

* ``dsqg_attention_v3(q, k, v, pos_bias, scale_embed)`` -- kernels/dsqg_attention_v3.py:445-456.
* ``dsqg_attention_v2(q, k, v, pos_bias)`` -- kernels/dsqg_attention_v2.py:417-428 (V3 with no
  scale_embed term).
* ``dsqg_attention_backend(q, k, v, pos_bias, scale_embed)`` -- the J=47 call of
  train/train_4096_13m_condU.py:104-105 (offset table chosen from pos_bias.shape[0]).
* ``dsqg_attention(...)`` -- the general form: any offset table, optional ``score_gain[H,J]``
  multiplying the content term and ``if_gain[H]`` multiplying the output (what
  train/train_2048_condU.py:187 does after the kernel), fused into the kernels.
* ``dsqg_attention_qkv(qkv, num_heads, ...)`` -- the same on the projection output
  qkv [B,N,3*H*HD] of train/train_2048_condU.py:169-175: the heads are read in place and the
  gradient comes back as one [B,N,3*H*HD] tensor.
* ``causal_mean_pool_gate(x, gate_pre)`` -- the interference pool of a DWARF block,
  train/train_2048_condU.py:289-292: ``sigmoid(gate_pre) * x.cumsum(1) / counts``.
* ``paged_kv_write`` / ``paged_decode_step`` / ``paged_kv_read`` and ``PagedKVCache`` -- full attention
  over a paged key/value cache, of the rows' type or 8 bits wide (no counterpart in the reference,
  whose full-attention layer, train/train_2048_condU.py:210-245, keeps no cache).
* ``window_attention`` -- full attention narrowed to a window and a few first positions, with gradients.
* ``paged_tree_step`` -- several drafted tokens of each sequence over that cache, as a tree or a chain, whole or within
  a window; ``draft_tree_accept`` -- which of the tokens drafted as a tree the model's picks keep.
* ``sample_tokens`` -- the next token from logits and given random numbers: the sampling of
  train/train_2048_condU.py:474-484 with top-k and min-p, in one kernel.

The output [B,H,N,HD] is stored token-major ([B,N,H,HD] memory), so the callers'
``out.permute(0, 2, 1, 3).reshape(B, N, H * HD)`` (train/train_2048_condU.py:186) is a view.

Dtype rules: bf16 in -> bf16 out with fp32 arithmetic; fp32 in -> fp32 out, computed in fp32
(the reference would downcast to bf16, kernels/dsqg_attention_v3.py:452-454); any other
float dtype (fp16 under autocast) is cast to bf16 and the result back, as the reference does.
Shape errors raise AssertionError, as the reference's asserts do (:363-365).
"""

from __future__ import annotations

from typing import Optional, Sequence, Union

import torch
from torch import Tensor

from . import _lib, ops
from .offsets import default_offsets, validate


def _check_shapes(q, k, v, pos_bias, scale_embed, score_gain, if_gain, offsets):
    assert q.dim() == 4, f"q must be [B,H,N,HD], got {tuple(q.shape)}"
    B, H, N, HD = q.shape
    assert k.shape == q.shape and v.shape == q.shape, "q, k, v must have the same shape"
    J = len(offsets)
    assert tuple(pos_bias.shape) == (J, H), f"pos_bias must be {(J, H)}, got {tuple(pos_bias.shape)}"
    if scale_embed is not None:
        assert tuple(scale_embed.shape) == (J, HD), \
            f"scale_embed must be {(J, HD)}, got {tuple(scale_embed.shape)}"
    if score_gain is not None:
        assert tuple(score_gain.shape) == (H, J), \
            f"score_gain must be {(H, J)}, got {tuple(score_gain.shape)}"
    if if_gain is not None:
        assert tuple(if_gain.shape) == (H,), f"if_gain must be {(H,)}, got {tuple(if_gain.shape)}"


def _f32(t: Optional[Tensor]) -> Optional[Tensor]:
    return None if t is None else t.float()


def _compute_dtype(q: Tensor, k: Tensor, v: Tensor):
    """q, k, v in the dtype the kernels compute in: q's if float32 or bfloat16, else bfloat16."""
    if q.dtype not in (torch.float32, torch.bfloat16):
        return q.bfloat16(), k.bfloat16(), v.bfloat16()
    return q, k.to(q.dtype), v.to(q.dtype)


def dsqg_attention(q: Tensor, k: Tensor, v: Tensor, pos_bias: Tensor,
                   scale_embed: Optional[Tensor] = None, *,
                   offsets: Optional[Sequence[int]] = None,
                   score_gain: Optional[Tensor] = None,
                   if_gain: Optional[Tensor] = None) -> Tensor:
    """DSQG attention over a fixed offset table (default chosen by pos_bias.shape[0]).

    q, k, v [B,H,N,HD]; pos_bias [J,H]; scale_embed [J,HD]; score_gain [H,J]; if_gain [H].
    Differentiable in q, k, v and every parameter.
    """
    if not ops.traced(q, k, v):
        return _lib.host().attention(q, k, v, pos_bias, scale_embed, score_gain, if_gain,
                                     default_offsets(pos_bias.shape[0]) if offsets is None
                                     else offsets)[0]
    offs = validate(offsets) if offsets is not None else default_offsets(pos_bias.shape[0])
    _check_shapes(q, k, v, pos_bias, scale_embed, score_gain, if_gain, offs)
    orig = q.dtype
    q, k, v = _compute_dtype(q, k, v)
    args = (q, k, v, pos_bias.float(), _f32(scale_embed), _f32(score_gain), _f32(if_gain),
            list(offs))
    out = ops.dsqg_fwd(*args)[0]
    return out if out.dtype == orig else out.to(orig)


def dsqg_attention_qkv(qkv: Tensor, num_heads: int, pos_bias: Tensor,
                       scale_embed: Optional[Tensor] = None, *,
                       offsets: Optional[Sequence[int]] = None,
                       score_gain: Optional[Tensor] = None,
                       if_gain: Optional[Tensor] = None,
                       kv_inject=None) -> Tensor:
    """dsqg_attention on q, k, v = the head views of qkv [B,N,3*H*HD] (the qkv_proj output).

    Same result as ``dsqg_attention(*split_qkv(qkv, num_heads), ...)``; differentiable in qkv
    and every parameter, with d(qkv) produced as one tensor.  ``kv_inject=(k_delta, v_delta)``
    ([B,H,N,HD] each) attends K + k_delta and V + v_delta (the Huygens injection of
    train/train_2048_condU.py:178-181); the deltas' gradients are the K / V slices of d(qkv).
    """
    assert qkv.dim() == 3, f"qkv must be [B,N,3*H*HD], got {tuple(qkv.shape)}"
    k_delta, v_delta = (None, None) if kv_inject is None else kv_inject
    if not ops.traced(qkv, *(() if kv_inject is None else (k_delta, v_delta))):
        return _lib.host().attention_qkv(qkv, num_heads, pos_bias, scale_embed, score_gain, if_gain,
                                         default_offsets(pos_bias.shape[0]) if offsets is None
                                         else offsets, k_delta, v_delta)
    offs = validate(offsets) if offsets is not None else default_offsets(pos_bias.shape[0])
    q, k, v = ops.split_qkv(qkv, num_heads)
    _check_shapes(q, k, v, pos_bias, scale_embed, score_gain, if_gain, offs)
    orig = qkv.dtype
    if orig not in (torch.float32, torch.bfloat16):
        qkv = qkv.bfloat16()
    params = (pos_bias.float(), _f32(scale_embed), _f32(score_gain), _f32(if_gain), list(offs))
    if kv_inject is None:
        out = ops.dsqg_fwd_qkv(qkv, num_heads, *params)[0]
    else:
        assert k_delta.shape == k.shape and v_delta.shape == v.shape, \
            f"kv_inject deltas must be {tuple(k.shape)}"
        out = ops.dsqg_fwd_qkv_kv(qkv, k_delta, v_delta, num_heads, *params)[0]
    return out if out.dtype == orig else out.to(orig)


def dsqg_attention_v3(q: Tensor, k: Tensor, v: Tensor, pos_bias: Tensor,
                      scale_embed: Tensor) -> Tensor:
    """Drop-in for kernels/dsqg_attention_v3.py:445 (44 offsets, Q-weighted scale term)."""
    return dsqg_attention(q, k, v, pos_bias, scale_embed)


def dsqg_attention_v2(q: Tensor, k: Tensor, v: Tensor, pos_bias: Tensor) -> Tensor:
    """Drop-in for kernels/dsqg_attention_v2.py:417 (44 offsets, no scale_embed)."""
    return dsqg_attention(q, k, v, pos_bias)


def dsqg_attention_backend(q: Tensor, k: Tensor, v: Tensor, pos_bias: Tensor,
                           scale_embed: Tensor) -> Tensor:
    """Drop-in for train/train_4096_13m_condU.py:104 (table by pos_bias.shape[0]: 44/46/47)."""
    return dsqg_attention(q, k, v, pos_bias, scale_embed)


def dsqg_attention_with_lse(q, k, v, pos_bias, scale_embed=None, *, offsets=None,
                            score_gain=None, if_gain=None):
    """(out, lse): out in the dtype rules above (differentiable), lse [B,H,N] fp32 (not)."""
    if not ops.traced(q, k, v):
        return _lib.host().attention(q, k, v, pos_bias, scale_embed, score_gain, if_gain,
                                     default_offsets(pos_bias.shape[0]) if offsets is None
                                     else offsets)
    offs = validate(offsets) if offsets is not None else default_offsets(pos_bias.shape[0])
    _check_shapes(q, k, v, pos_bias, scale_embed, score_gain, if_gain, offs)
    orig = q.dtype
    q, k, v = _compute_dtype(q, k, v)
    args = (q, k, v, pos_bias.float(), _f32(scale_embed), _f32(score_gain), _f32(if_gain),
            list(offs))
    out, lse = ops.dsqg_fwd(*args)[:2]
    return (out if out.dtype == orig else out.to(orig)), lse


def dsqg_decode_step(q: Tensor, k_new: Tensor, v_new: Tensor, k_ring: Tensor, v_ring: Tensor,
                     pos: Tensor, pos_bias: Tensor, scale_embed: Optional[Tensor] = None, *,
                     offsets: Optional[Sequence[int]] = None,
                     score_gain: Optional[Tensor] = None,
                     if_gain: Optional[Tensor] = None) -> Tensor:
    """One decode step: q/k_new/v_new [B,H,D], rings [B,H,S,D] (updated in place), pos [B]."""
    rows = (q, k_new, v_new, k_ring, v_ring)
    # (The step has no gradient; the custom op is what says so when one is asked for.)
    if not ops.traced(*rows, pos) and not (torch.is_grad_enabled() and any(t.requires_grad for t in rows)):
        return _lib.host().decode(*rows, pos, pos_bias, scale_embed, score_gain, if_gain,
                                  default_offsets(pos_bias.shape[0]) if offsets is None else offsets)
    offs = validate(offsets) if offsets is not None else default_offsets(pos_bias.shape[0])

    def f32(t):
        return None if t is None else t.detach().float().contiguous()

    return ops.dsqg_decode(q.contiguous(), k_new.contiguous(), v_new.contiguous(), k_ring,
                           v_ring, pos.to(torch.int64).contiguous(), f32(pos_bias),
                           f32(scale_embed), f32(score_gain), f32(if_gain), list(offs))


def causal_mean_pool_gate(x: Tensor, gate_pre: Tensor) -> Tensor:
    """``sigmoid(gate_pre) * x.cumsum(1) / (n + 1)`` over [B,N,C] (C a multiple of 8), forward
    and backward on the HIP scan kernels: the interference pool of train/train_2048_condU.py:
    289-292 (``pool = xi.cumsum(dim=1) / counts``; ``inter = sigmoid(inter_gate(xi)) * pool``).

    x and gate_pre may be float32, bfloat16 or float16 and may differ (under autocast the
    reference has a float32 LayerNorm output and a float16 gate); the result has their promoted
    dtype, as the reference's product does, and the sigmoid is rounded to gate_pre's dtype first,
    as torch's sigmoid of that tensor is.  Sums are fp32 and deterministic.
    """
    assert x.dim() == 3, f"x must be [B,N,C], got {tuple(x.shape)}"
    assert gate_pre.shape == x.shape, (f"gate_pre must match x {tuple(x.shape)}, "
                                       f"got {tuple(gate_pre.shape)}")
    assert x.shape[2] % 8 == 0, f"channel count {x.shape[2]} must be a multiple of 8"
    if ops.traced(x, gate_pre):
        return ops.pool_gate_fwd(x, gate_pre)
    return _lib.host().pool_gate(x, gate_pre)


def window_attention(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int = 0, *,
                     lengths: Optional[Tensor] = None, softmax_scale: Optional[float] = None) -> Tensor:
    """Causal softmax attention within a window, forward and backward on the HIP kernels: position i of q [B,H,N,D] sees
    position j <= i of k, v [B,Hkv,N,D] if i - j < window or j < sinks, query head h the key/value head h // (H // Hkv);
    returns out [B,H,N,D] (token-major storage).  A window of N or more is full causal attention.

    With lengths [B], integers, rows from lengths[b] on are not there: nothing sees them, their outputs and gradients
    are zeros.  softmax_scale defaults to D ** -0.5.  float32, bfloat16 and float16, head dims 32, 64, 80, 96 and 128;
    sums and softmax statistics are fp32 and deterministic, and weights (in the backward their gradients too) are
    rounded once to a 16-bit type before they multiply rows.  What a query does not see does not reach it, whatever
    it holds.  Outputs are finite where the values are, up to 2^-7 below the type's largest.  A training pass in 16 bits keeps,
    beside out, as much again for what its rounding took off, which the gradients need.  There is no second derivative.
    ``paged_tree_step`` with the same window and sinks continues over a cache.
    """
    if ops.traced(q, k, v):
        return ops.window_fwd(q, k, v, lengths, window, sinks, softmax_scale)[0]
    return _lib.host().window(q, k, v, lengths, window, sinks, softmax_scale)


def paged_kv_write(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, pos: Tensor, *,
                   counts: Optional[Tensor] = None, rows: Optional[Tensor] = None,
                   k_scale: Optional[Tensor] = None, v_scale: Optional[Tensor] = None) -> None:
    """Write row i of each sequence of k and v [B,Hkv,N,D] to position pos[b] + i of a paged cache, for
    i < counts[b] (default: all N); every other row of the pages stays as it is.  With rows [B,M], integers, row
    rows[b,i] goes to position pos[b] + i instead, for i < M; a number that is no row of k and v writes nothing
    (``draft_tree_accept`` returns such paths).

    k_pages, v_pages [P,Hkv,page,D] are pools of pages (page a power of two from 16) and page_table [B,M]
    int32 names the page that holds positions page * j .. page * (j + 1) - 1 of each sequence.  Rows are
    float32, bfloat16 or float16, and so are the pages, of the same type, or they are 8 bits wide
    (float8_e4m3fn or int8) with k_scale, v_scale [P,Hkv,page] float8_e8m0fnu: a row's scale is the
    smallest power of two that brings its largest magnitude to at most 448 or 127, and its values are
    rounded once.  A row that holds an infinity or NaN reads as NaN from 8-bit pages.  Positions without
    a page (a number that is none of the pool's, a position past the table) are not written.  Sequences may
    share pages that none of them writes; a page that two of them write, or rows that are views of the pages
    themselves, have no defined result.  No gradient passes through the cache.
    """
    if ops.traced(k, v, k_pages, v_pages):
        if rows is not None:
            return ops.paged_kv_write_rows(k, v, k_pages, v_pages, page_table, pos, counts, rows, k_scale, v_scale)
        return ops.paged_kv_write(k, v, k_pages, v_pages, page_table, pos, counts, k_scale, v_scale)
    return _lib.host().paged_write(k, v, k_pages, v_pages, page_table, pos, counts, rows, k_scale, v_scale)


def paged_kv_read(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor,
                  max_len: Optional[int] = None, *, k_scale: Optional[Tensor] = None,
                  v_scale: Optional[Tensor] = None, dtype: Optional[torch.dtype] = None):
    """(k, v) [B,Hkv,max_len,D]: positions 0 .. lengths[b] - 1 of each sequence of a paged cache (see
    ``paged_kv_write``), zeros behind them, NaN at a position without a page.  max_len defaults to the
    table's positions, dtype to the pages' or, for 8-bit pages, bfloat16 (whose precision holds their values)."""
    if max_len is None:
        max_len = page_table.shape[1] * k_pages.shape[2]
    if dtype is None:
        dtype = torch.bfloat16 if k_pages.element_size() == 1 else k_pages.dtype
    if ops.traced(k_pages, v_pages, page_table):
        return ops.paged_kv_read(k_pages, v_pages, page_table, lengths, max_len, dtype, k_scale, v_scale)
    return _lib.host().paged_read(k_pages, v_pages, page_table, lengths, max_len, dtype, k_scale, v_scale)


def paged_decode_step(q: Tensor, k_new: Optional[Tensor], v_new: Optional[Tensor], k_pages: Tensor,
                      v_pages: Tensor, page_table: Tensor, pos: Tensor, *, k_scale: Optional[Tensor] = None,
                      v_scale: Optional[Tensor] = None, softmax_scale: Optional[float] = None) -> Tensor:
    """One decode step over a paged cache (see ``paged_kv_write``): k_new, v_new [B,Hkv,D] go to position
    pos[b], and the H = Hkv * G query heads q [B,H,D] attend positions 0 .. pos[b] (query head h the
    key/value head h // G); returns out [B,H,D].

    softmax_scale defaults to D ** -0.5.  With k_new = v_new = None nothing is written and position
    pos[b] is attended as the pages hold it.  A sequence with pos[b] < 0 attends nothing and gets zeros;
    one that attends a position without a page gets NaN.  Sums are fp32 and the result does not change
    from call to call.  Values below 2^-90 (8-bit rows: whose largest is below 2^-70) lose bits or vanish, a
    row of less than 2^-96 of the heaviest one's weight weighs nothing (an infinite value there gives NaN), and
    queries over 8-bit pages must be below 2^112.  The step has no gradient.
    """
    if ops.traced(q, k_pages, v_pages):
        return ops.paged_decode(q, k_new, v_new, k_pages, v_pages, page_table, pos, k_scale, v_scale, softmax_scale)
    return _lib.host().paged_decode(q, k_new, v_new, k_pages, v_pages, page_table, pos, k_scale, v_scale,
                                    softmax_scale)


def paged_tree_step(q: Tensor, k_new: Optional[Tensor], v_new: Optional[Tensor], k_pages: Tensor, v_pages: Tensor,
                    page_table: Tensor, pos: Tensor, parents: Optional[Tensor] = None, *,
                    counts: Optional[Tensor] = None, window: Optional[int] = None, sinks: int = 0,
                    k_scale: Optional[Tensor] = None, v_scale: Optional[Tensor] = None,
                    softmax_scale: Optional[float] = None) -> Tensor:
    """A step of T tokens of each sequence, drafted as a tree, over a paged cache (see ``paged_kv_write``): k_new, v_new
    [B,Hkv,T,D] go to positions pos[b] .. pos[b] + T - 1, and node i of the H = Hkv * G query heads q [B,H,T,D] attends
    the positions before pos[b], its ancestors and itself; returns out [B,H,T,D] (token-major storage).  T is at most 64.

    Node i hangs on the earlier node parents[i] (or parents[b,i]) or, -1, on the last position before pos[b]; without
    parents the tokens are a chain.  With counts, sequence b has counts[b] nodes; rows behind them are not written.
    What is no node, behind counts[b] or on parents that do not lead over earlier nodes to -1, gets zeros.  With a window
    a node, at the place pos[b] + its depth, sees the window places up to its own and those below ``sinks``
    (``window_attention``); a chain of one token is a windowed layer's decode step, and pages that no later
    step sees may be given away.

    With k_new = v_new = None nothing is written and the draft's rows are attended as the pages hold them.  A
    sequence with pos[b] < 0 gets zeros and writes nothing, a node that sees a position without a page NaN.  A row that a
    node does not see does not reach it, whatever it holds.  The range of values is ``paged_decode_step``'s.  Weights of
    T * G > 16 tokens and heads are rounded once, to the cache's 16-bit type (8 bits: bfloat16; not with float16
    queries, which keep two terms), before they multiply the values.  The step has no gradient.  ``draft_tree_accept`` says which rows to keep.
    """
    if ops.traced(q, k_pages, v_pages):
        return ops.paged_tree(q, k_new, v_new, k_pages, v_pages, page_table, pos, parents, counts, window, sinks, k_scale,
                              v_scale, softmax_scale)
    return _lib.host().paged_tree(q, k_new, v_new, k_pages, v_pages, page_table, pos, parents, counts, window, sinks,
                                  k_scale, v_scale, softmax_scale)


def draft_tree_accept(tokens: Tensor, parents: Tensor, picks: Tensor, counts: Optional[Tensor] = None):
    """(path [B,T], n [B], next [B]), int64: which of the tokens drafted as a tree are kept.

    Node i of sequence b has the token tokens[b,i] and hangs on the node parents[i] (or parents[b,i]); picks[b,i] is
    what the model chose after it.  Node 0, the token that was certain before, is kept; from a node the walk goes to its
    first child behind it whose token is the node's pick.  path lists the nodes on the way, -1 behind them, n counts
    them, and next is the pick after the last: the next draft's node 0.  With counts, sequence b has counts[b] nodes (of
    none: n 0 and next -1).  T is at most 64.  ``paged_kv_write(..., counts=n, rows=path)`` keeps their rows.
    """
    if ops.traced(tokens, parents, picks):
        return ops.tree_accept(tokens, parents, picks, counts)
    return _lib.host().tree_accept(tokens, parents, picks, counts)


def sample_tokens(logits: Tensor, u: Tensor, temperature: Union[float, Tensor] = 1.0, top_k: Union[int, Tensor] = 0,
                  top_p: Union[float, Tensor] = 1.0, min_p: Union[float, Tensor] = 0.0, *,
                  return_logprobs: bool = False):
    """Tokens [...] (int64) drawn from logits [...,V] with one number u [...] from [0, 1) for each row; with
    ``return_logprobs`` also the log probabilities (float32) that they were drawn with.

    Weights are exp((x - max x) / temperature).  In the order of x, the largest first and of equal ones the lower
    index, the tokens that stay are the first top_k, of those the ones before which at most top_p of their mass
    lies (train/train_2048_condU.py:478-482), of those the ones of at least min_p of the largest weight; the drawn one
    is the first, by index, whose running mass is above u times the mass that stays.  top_k = 0, top_p = 1 and min_p
    = 0 limit nothing; temperature 0 takes the largest logit (the first of equal ones, log probability 0).  Each
    setting is a number or a tensor of one for each row, where values past a limit's range mean its end (a
    temperature that is not above 0 is 0) and a NaN no limit.  A NaN logit is no candidate, as -infinity is; a
    row without candidates gives -1 and -infinity.  Masses are summed as whole numbers: the result depends on nothing but
    the row.  Nothing here has a gradient.
    """
    def split(x, none):
        return (none, x) if isinstance(x, Tensor) else (x, None)

    (t, ts), (k, ks), (p, ps), (m, ms) = split(temperature, 1.0), split(top_k, 0), split(top_p, 1.0), split(min_p, 0.0)
    fn = ops.sample_tokens if ops.traced(logits, u) else _lib.host().sample
    tokens, logprobs = fn(logits, u, t, k, p, m, ts, ks, ps, ms, return_logprobs)
    return (tokens, logprobs) if return_logprobs else tokens


class DSQGRingCache:
    """Per-layer O(1) decode cache: K/V rings of S = max(offset)+1 slots (README.md:175-179).

    ``prefill(k, v)`` loads the last S positions of a prompt (k, v [B,H,N,D]); ``step(q, k_t,
    v_t)`` runs one decode step at the current position and advances it.
    """

    def __init__(self, B: int, H: int, D: int, offsets: Sequence[int], dtype=torch.bfloat16,
                 device="cuda", slots: Optional[int] = None):
        self.offsets = validate(offsets)
        self.S = int(slots) if slots is not None else self.offsets[-1] + 1
        assert self.S > self.offsets[-1], "ring needs at least max(offset)+1 slots"
        self.k_ring = torch.zeros((B, H, self.S, D), dtype=dtype, device=device)
        self.v_ring = torch.zeros_like(self.k_ring)
        self.pos = torch.zeros((B,), dtype=torch.int64, device=device)

    def prefill(self, k: Tensor, v: Tensor) -> None:
        """Write prompt rows m = N-S..N-1 (those that exist) to slots m mod S; pos becomes N."""
        B, H, N, D = k.shape
        state = (self.k_ring, self.v_ring, self.pos)
        if self.k_ring.is_cuda and not ops.traced(k, v, *state) \
                and self.S == self.k_ring.shape[2] and _lib.host().ring_load(k, v, *state):
            return
        lo = max(0, N - self.S)
        idx = torch.arange(lo, N, device=k.device)
        self.k_ring[:, :, idx % self.S] = k[:, :, lo:N].to(self.k_ring.dtype)
        self.v_ring[:, :, idx % self.S] = v[:, :, lo:N].to(self.v_ring.dtype)
        self.pos.fill_(N)

    def step(self, q: Tensor, k_new: Tensor, v_new: Tensor, pos_bias: Tensor,
             scale_embed: Optional[Tensor] = None, score_gain: Optional[Tensor] = None,
             if_gain: Optional[Tensor] = None) -> Tensor:
        out = dsqg_decode_step(q, k_new, v_new, self.k_ring, self.v_ring, self.pos, pos_bias,
                               scale_embed, offsets=self.offsets, score_gain=score_gain,
                               if_gain=if_gain)
        self.pos += 1
        return out


class PagedKVCache:
    """Key/value cache of one full-attention layer for B sequences of up to ``max_len`` positions, in pages
    (see ``paged_kv_write``), each sequence at a position of its own (``pos`` [B], on the device).

    ``dtype`` is the type of the rows and, unless ``kv_dtype`` (torch.float8_e4m3fn or torch.int8) asks for
    8 bits, of the pages.  ``prefill(k, v)`` loads a prompt, ``write(k, v)`` appends rows, ``step(q, k_t,
    v_t)`` runs one decode step and advances, ``tree_step`` and ``accept`` try several drafted tokens and keep some of
    them, ``read()`` returns the rows.  Every sequence owns its pages,
    sequence b those from b * M on; a caller that shares or moves pages sets ``page_table``.  The host
    does not know the positions: rows past a sequence's last page are not kept, and its steps give NaN.
    A sequence at a negative position is not in use: its pages and position stay as they are and its steps
    give zeros, until ``pos`` is set again.
    """

    def __init__(self, B: int, H: int, D: int, max_len: int, dtype=torch.bfloat16, device="cuda",
                 kv_dtype: Optional[torch.dtype] = None, page_size: int = 64):
        assert max_len >= 1, f"max_len must be positive, got {max_len}"
        assert D in _lib.supported_head_dims(), f"head dim {D} is none of {_lib.supported_head_dims()}"
        assert kv_dtype in (None, dtype, torch.float8_e4m3fn, torch.int8), \
            f"kv_dtype must be float8_e4m3fn, int8 or the rows' {dtype}, got {kv_dtype}"
        self.dtype = dtype
        self.max_len = int(max_len)
        M = -(-self.max_len // page_size)
        shape = (B * M, H, page_size, D)
        kv = kv_dtype or dtype
        self.k_pages = torch.zeros(shape, dtype=kv, device=device)
        self.v_pages = torch.zeros_like(self.k_pages)
        self.k_scale = self.v_scale = None
        if self.k_pages.element_size() == 1:
            self.k_scale = torch.zeros(shape[:3], dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
            self.v_scale = torch.zeros_like(self.k_scale)
        self.page_table = torch.arange(B * M, dtype=torch.int32, device=device).view(B, M)
        self.pos = torch.zeros((B,), dtype=torch.int64, device=device)

    def _state(self):
        return dict(k_scale=self.k_scale, v_scale=self.v_scale)

    def prefill(self, k: Tensor, v: Tensor, counts: Optional[Tensor] = None) -> None:
        """Write prompts k, v [B,H,N,D] from position 0 on, counts[b] rows of each (default: N); pos becomes
        that."""
        assert k.shape[2] <= self.max_len, f"prompt of {k.shape[2]} rows exceeds the cache ({self.max_len})"
        counts = self._write(k, v, torch.zeros_like(self.pos), counts)
        if counts is None:
            self.pos.fill_(k.shape[2])
        else:
            self.pos.copy_(counts)

    def write(self, k: Tensor, v: Tensor, counts: Optional[Tensor] = None) -> None:
        """Append rows k, v [B,H,N,D], counts[b] of each (default: N), and advance."""
        used = self.pos >= 0
        counts = used * (k.shape[2] if counts is None else counts)
        self.pos += self._write(k, v, self.pos, counts)

    def _write(self, k: Tensor, v: Tensor, pos: Tensor, counts: Optional[Tensor]) -> Optional[Tensor]:
        if counts is not None:
            assert not (counts.is_floating_point() or counts.is_complex() or counts.dtype == torch.bool), \
                f"counts must be integers, got {counts.dtype}"
            # (As int64: a narrow type may not hold the number of rows that they are limited to.)
            counts = counts.long().clamp(0, k.shape[2])
        paged_kv_write(k.detach().to(self.dtype), v.detach().to(self.dtype), self.k_pages, self.v_pages,
                       self.page_table, pos, counts=counts, **self._state())
        return counts

    def step(self, q: Tensor, k_new: Tensor, v_new: Tensor, softmax_scale: Optional[float] = None,
             window: Optional[int] = None, sinks: int = 0) -> Tensor:
        """Output [B,H*G,D] of one new token per sequence at its position, which advances.  With a window it sees the
        last ``window`` positions, its own among them, and those below ``sinks``."""
        if window is not None:
            out = self.tree_step(q.unsqueeze(2), k_new.unsqueeze(2), v_new.unsqueeze(2), window=window, sinks=sinks,
                                 softmax_scale=softmax_scale)[:, :, 0]
            self.pos += self.pos >= 0
            return out
        dt = self.dtype
        out = paged_decode_step(q.detach().to(dt), k_new.detach().to(dt), v_new.detach().to(dt), self.k_pages,
                                self.v_pages, self.page_table, self.pos, softmax_scale=softmax_scale,
                                **self._state())
        self.pos += self.pos >= 0
        return out.to(q.dtype)

    def tree_step(self, q: Tensor, k_new: Tensor, v_new: Tensor, parents: Optional[Tensor] = None,
                  counts: Optional[Tensor] = None, window: Optional[int] = None, sinks: int = 0,
                  softmax_scale: Optional[float] = None) -> Tensor:
        """Output [B,H*G,T,D] of T tokens drafted as a tree (``paged_tree_step``).  Their rows lie behind the sequences'
        positions, which stay as they are until ``accept`` says what is kept."""
        dt = self.dtype
        out = paged_tree_step(q.detach().to(dt), k_new.detach().to(dt), v_new.detach().to(dt), self.k_pages, self.v_pages,
                              self.page_table, self.pos, parents, counts=counts, window=window, sinks=sinks,
                              softmax_scale=softmax_scale, **self._state())
        return out.to(q.dtype)

    def accept(self, k_new: Tensor, v_new: Tensor, path: Tensor, n: Tensor) -> None:
        """Keep the rows of the nodes path[b,:n[b]] (``draft_tree_accept``) of a draft's k_new, v_new, and advance by n."""
        n = (self.pos >= 0) * n.long().clamp(0, path.shape[1])
        paged_kv_write(k_new.detach().to(self.dtype), v_new.detach().to(self.dtype), self.k_pages, self.v_pages,
                       self.page_table, self.pos, counts=n, rows=path, **self._state())
        self.pos += n

    def read(self, max_len: Optional[int] = None, dtype: Optional[torch.dtype] = None):
        """(k, v) [B,H,max_len,D] (default: the cache's max_len) of the positions written so far, zeros
        behind them, in the rows' dtype or another."""
        return paged_kv_read(self.k_pages, self.v_pages, self.page_table, self.pos,
                             self.max_len if max_len is None else max_len, dtype=dtype or self.dtype,
                             **self._state())
