"""Plain restatement of the paged key/value cache on the CPU, in 64 bits (test infrastructure only).

Written from the definition in include/dsqg.h: rows of a sequence by position through a page table, rows
of 8-bit pools as code * 2^(byte - 127), one query row's softmax attention over them.
"""

import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def encode_row(row, kv_dtype):
    """(codes as floats, byte) of one row of Python floats."""
    top = LARGEST[kv_dtype]
    if not all(math.isfinite(x) for x in row):
        return [0.0] * len(row), 255
    size = max(abs(x) for x in row)
    e = -127
    if size > 0:
        e = max(-127, math.frexp(size)[1] - 12)
        while size > math.ldexp(top, e):
            e += 1
    codes = []
    for x in row:
        y = math.ldexp(x, -e)
        step = 1.0
        if kv_dtype == torch.float8_e4m3fn:
            lead = math.frexp(abs(y))[1] - 1 if y else -6
            step = math.ldexp(1.0, max(lead, -6) - 3)
        codes.append(math.copysign(round(y / step) * step, y))  # Python's round: ties to even, no sign of zero
    return codes, e + 127


def encode(x, kv_dtype):
    """(codes, bytes): the stored form of rows x [..., D], codes as float64."""
    rows = [encode_row(r, kv_dtype) for r in x.double().reshape(-1, x.shape[-1]).tolist()]
    codes = torch.tensor([r[0] for r in rows], dtype=torch.float64).reshape(x.shape)
    return codes, torch.tensor([r[1] for r in rows], dtype=torch.uint8).reshape(x.shape[:-1])


def values(pages, scale=None):
    """What a pool's rows stand for, float64."""
    x = pages.double()
    if scale is None:
        return x
    e = scale.view(torch.uint8).double()
    return torch.where((e == 255)[..., None], torch.full_like(x, math.nan), x * (2.0 ** (e - 127))[..., None])


def sequence(pages, table, b, length, scale=None):
    """Rows 0 .. length - 1 of sequence b, [H, length, D] float64; NaN where there is no page."""
    P, H, page, D = pages.shape
    out = torch.full((H, length, D), math.nan, dtype=torch.float64)
    for j in range(min(table.shape[1], -(-length // page))):
        i, n = int(table[b, j]), min(page, length - j * page)
        if 0 <= i < P:
            out[:, j * page:j * page + n] = values(pages[i, :, :n], None if scale is None else scale[i, :, :n])
    return out


def attend(q, k, v, scale):
    """(out, mass, size) of q [H, D] over k, v [Hkv, T, D]: out [H, D] and, for a bound on a 32-bit
    evaluation, mass [H, 2, D], sum_t w_t |v_t| and sum_t |v_t|, and size [H, 1], the largest
    |scale| * sum_i |q_i k_ti|."""
    H, G = q.shape[0], q.shape[0] // k.shape[0]
    out, mass, size = [], [], []
    for h in range(H):
        kk, vv, x = k[h // G], v[h // G], q[h].double()
        s = kk @ x * scale
        w = torch.exp(s - s.max()) if len(s) else s
        w = w / w.sum()
        out.append(w @ vv)
        mass.append(torch.stack([w @ vv.abs(), vv.abs().sum(0)]))
        size.append((kk.abs() @ x.abs()).max() * abs(scale))
    return torch.stack(out), torch.stack(mass), torch.stack(size)[:, None]


def bound(out, mass, size, D, T, dtype):
    """How far a kernel's out may be from the exact one, element by element, u = 2^-24.

    A score's D products and its scaling: (D + 3) u of ``size`` at most, D u of it from the sum and the
    rest from the factor, its conversion to base 2 and the difference to the maximum (whose magnitude is at
    most twice ``size``: 4 u more); 2^x itself: 2 u.  A weight is so far off relative to itself, and the
    normalised one twice that.  The sums over T rows: T u each, twice; joining parts: a few roundings each,
    16 u.  All of these are relative to ``mass[:, 0]``.  A weight, or its product with the factor that a
    larger maximum brings, that lies below the normal numbers may come out as zero, which three such
    products in turn (tile, wave, chunk) add up to 4 * 2^-96 for each row, as the largest weight is 2^-30:
    that much of ``mass[:, 1]``.  Weights that enter a product in two 16-bit terms are 2^-16 off in bfloat16
    (a term of 8 bits rounded down and one of 8 bits rounded: 2^-7 * 2^-9) and, in float16, 2^-21 (2^-10 *
    2^-11) or its subnormal step where the largest weight is 2^14: 2 * 2^-38 of ``mass[:, 1]`` (a float32
    kernel has no such terms; its results' bound leaves them out).  Last, the result's rounding to its type, half a step of it: eps / 2
    relative, or half the smallest subnormal.
    """
    u = 2.0 ** -24
    w = 2 * ((D + 7) * u * size + 2 * u)
    tol = mass[:, 0] * (w + (2 * T + 16) * u) + mass[:, 1] * 4 * 2.0 ** -96
    if dtype != torch.float32:
        tol = tol + mass[:, 0] * 2.0 ** -16 + (mass[:, 1] * 2.0 ** -37 if dtype == torch.float16 else 0)
    fi = torch.finfo(dtype)
    return tol + (out.abs() + tol) * (fi.eps / 2) + fi.smallest_normal * fi.eps
