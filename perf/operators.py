"""Performance cases of the paged key/value cache: its decode step, writing prompts into it, reading
it back.

A pool of pages [P, Hkv, page, D] holds the keys of all sequences of one layer, another one the
values; ``page_table`` [B, M] says which page holds positions ``page * j .. page * (j + 1) - 1`` of a
sequence.  A pool is float32, bfloat16 or float16, or 8 bits wide (``float8_e4m3fn`` or ``int8``)
with one power-of-two scale for each row of D values (``float8_e8m0fnu`` [P, Hkv, page]): the
smallest power of two that brings the row's largest magnitude to at most the type's largest value.

* step:  the new token's key and value row go to position ``pos`` of each sequence, and its H = Hkv *
  G query heads attend positions 0 .. pos;
* write: N rows of each sequence go to positions pos .. pos + count - 1 (an 8-bit pool is then read
  back, as the next stretch of a prompt that is taken in pieces does);
* read:  positions 0 .. length - 1 of each sequence come back as one tensor, zeros behind them.

``own`` chooses between the framework's kernels and the same mathematics in elementary torch
operations.  Steps write the same rows into the same places each time, so they can be repeated.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}


def _case(name, op, B, Hkv, G, D, T, page, dtype, cache, ragged=False, N=0):
    return dict(name=name, op=op, B=B, Hkv=Hkv, G=G, D=D, T=T, page=page, dtype=dtype, cache=cache,
                ragged=ragged, N=N)


def listed():
    return [
        # One chat-sized sequence of the 13M model's layer: the smallest call, where latency counts.
        _case("step_77", "step", 1, 8, 1, 32, 77, 64, "bf16", "bf16"),
        # The same layer in float32, four sequences up to the position table's end.
        _case("step_13m_f32", "step", 4, 8, 1, 32, 2048, 64, "f32", "f32", ragged=True),
        # Batched serving of the 85M model's layer, sequences of many lengths in small pages.
        _case("step_85m_batch", "step", 32, 12, 1, 64, 2048, 16, "bf16", "bf16", ragged=True),
        # One long document: eight heads have to fill the chip.
        _case("step_long", "step", 1, 8, 1, 64, 131072, 256, "bf16", "bf16"),
        # Shared key/value heads over an 8-bit cache, a full batch of long sequences: the largest.
        _case("step_shared_e4m3", "step", 64, 8, 4, 128, 8192, 64, "bf16", "e4m3", ragged=True),
        # Odd counts of sequences, heads and positions, float16 queries, integer cache.
        _case("step_odd_int8", "step", 5, 3, 5, 80, 5001, 32, "f16", "int8", ragged=True),
        # One key/value head for all query heads.
        _case("step_one_kv_head", "step", 16, 1, 8, 96, 16001, 128, "bf16", "bf16", ragged=True),
        # A chat-sized prompt into an empty cache: launches and host work.
        _case("write_77", "write", 1, 8, 1, 32, 77, 64, "bf16", "bf16", N=77),
        # A batch of whole prompts of the 85M model into an 8-bit cache, and the cache read back.
        _case("write_85m_e4m3", "write", 8, 12, 1, 64, 2048, 64, "bf16", "e4m3", N=2048),
        # The last stretch of ragged prompts, an odd number of rows, and the whole prefix read back.
        _case("write_ragged_int8", "write", 16, 8, 1, 128, 4096, 16, "f16", "int8", ragged=True, N=1023),
        # A small float32 cache, ragged: what a check or an export reads.
        _case("read_f32", "read", 4, 8, 1, 32, 2047, 64, "f32", "f32", ragged=True),
        # Two long sequences out of an 8-bit cache.
        _case("read_long_e4m3", "read", 2, 8, 1, 128, 65536, 256, "bf16", "e4m3"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "step", "step", "step", "write", "read"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    cache = rng.choice([dtype, dtype, "e4m3", "int8"])
    page = rng.choice([16, 32, 64, 128, 256])
    while True:
        B, Hkv, D, T = _log_int(rng, 1, 64), _log_int(rng, 1, 16), rng.choice([32, 64, 80, 96, 128]), \
            _log_int(rng, 1, 131072)
        # A step costs its cache; the others move it out again at two to four bytes a value.
        if B * Hkv * D * T * SIZES[cache] <= (1 << 28 if op == "step" else 1 << 25):
            break
    G = rng.choice([1, 1, 2, 3, 4, 5, 6, 8, 16]) if op == "step" else 1
    return dict(op=op, B=B, Hkv=Hkv, G=G, D=D, T=T, page=page, dtype=dtype, cache=cache,
                ragged=rng.random() < 0.6, N=_log_int(rng, 1, T) if op == "write" else 0)


def _lengths(c):
    """Positions in use of each sequence: all T, or spread from T down to a quarter of it, the last of
    three or more a single one (a request that has just come in), in an order of no rule."""
    B, T = c["B"], c["T"]
    if not c["ragged"]:
        return [T] * B
    n = [max(1, T - (3 * T * i) // (4 * B)) for i in range(B)]
    if B > 2:
        n[-1] = 1
    random.Random(B * 1000003 + T).shuffle(n)
    return n


def _counts(c):
    """Rows that a write brings to each sequence: the last of its positions, N at most."""
    return [min(c["N"], n) for n in _lengths(c)]


def _quantise(x, cache):
    """Rows of x as the 8-bit values' bytes and the scales' exponent bytes."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    # 448 = 0.875 * 2^9 and 127 = 0.9921875 * 2^7 are the types' largest values.
    e = e - 9 + (m > 0.875).int() if cache == "e4m3" else e - 7 + (m > 0.9921875).int()
    e = torch.where(m == 0, -127, e.clamp(min=-127))
    # 2^-e by its bits: the chip's pow may be off in the last one.
    y = x * ((127 - e) << 23).to(torch.int32).view(torch.float32)[..., None]
    y = y.to(torch.float8_e4m3fn) if cache == "e4m3" else y.round().to(torch.int8)
    return y.view(torch.uint8), (e + 127).to(torch.uint8)


def _values(pages, scale):
    """What a pool's rows stand for, in float32."""
    x = pages.float()
    return x if scale is None else x * scale.float()[..., None]


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, Hkv, G, D, T, page = c["B"], c["Hkv"], c["G"], c["D"], c["T"], c["page"]
    dt, ct = DTYPES[c["dtype"]], DTYPES[c["cache"]]
    n = _lengths(c)
    used = [-(-x // page) for x in n]
    M = -(-T // page)
    P = sum(used) + 2  # two pages that belong to nobody

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    # Keys differ in size from channel to channel, as those of trained models do.
    channel = torch.exp(0.5 * randn(D))

    def pool(ch):
        x = randn(P, Hkv, page, D) * ch
        if SIZES[c["cache"]] > 1:
            return x.to(ct), None
        y, e = _quantise(x, c["cache"])
        return y.view(ct), e.view(torch.float8_e8m0fnu)

    s = dict(case=c)
    s["k_pages"], s["k_scale"] = pool(channel)
    s["v_pages"], s["v_scale"] = pool(1.0)
    # Pages in an order of no rule; entries behind a sequence's last page name none.
    order = torch.randperm(P, generator=g, device=DEV)[:sum(used)].to(torch.int32).cpu()
    table = torch.full((B, M), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    s["page_table"] = table.to(DEV)
    s["lengths"] = torch.tensor(n, dtype=torch.int64, device=DEV)
    if c["op"] == "step":
        s["q"] = (randn(B, Hkv * G, D) * 1.5).to(dt)
        s["k"], s["v"] = (randn(B, Hkv, D) * channel).to(dt), randn(B, Hkv, D).to(dt)
        s["pos"] = s["lengths"] - 1
    elif c["op"] == "write":
        # Head views of a projection's output.
        N = c["N"]
        kv = randn(B, N, 2, Hkv, D)
        kv[:, :, 0] *= channel
        kv = kv.to(dt)
        s["k"], s["v"] = (kv[:, :, i].permute(0, 2, 1, 3) for i in (0, 1))
        s["counts"] = torch.tensor(_counts(c), dtype=torch.int64, device=DEV)
        s["pos"] = s["lengths"] - s["counts"]
    return s


# ---- The framework's calls. ------------------------------------------------------------------

def _own_step(s):
    import dwarf_amd
    return dwarf_amd.paged_decode_step(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"],
                                       s["pos"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_write(s):
    import dwarf_amd
    dwarf_amd.paged_kv_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["pos"],
                             counts=s["counts"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_read(s):
    import dwarf_amd
    return dwarf_amd.paged_kv_read(s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["case"]["T"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"], dtype=DTYPES[s["case"]["dtype"]])


# ---- The same in elementary operations. --------------------------------------------------------

def _put(pages, scale, ids, slots, rows, cache):
    """rows [n, Hkv, D] to the slots of the pages."""
    if scale is None:
        pages[ids, :, slots] = rows.to(pages.dtype)
        return
    y, e = _quantise(rows, cache)
    pages.view(torch.uint8)[ids, :, slots] = y
    scale.view(torch.uint8)[ids, :, slots] = e


def _gather(pages, scale, table):
    """The values of every position of the table, [B, Hkv, M * page, D] float32."""
    B, M = table.shape
    at = table.clamp(min=0).long()
    _, H, page, D = pages.shape
    x = pages.view(torch.uint8)[at].view(pages.dtype) if scale is not None else pages[at]
    x = _values(x, None if scale is None else scale.view(torch.uint8)[at].view(scale.dtype))
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, M * page, D)


def _plain_step(s):
    c, q = s["case"], s["q"]
    B, H, D = q.shape
    page = c["page"]
    pos, table = s["pos"], s["page_table"]
    ids, slots = table.gather(1, (pos // page)[:, None])[:, 0].long(), pos % page
    _put(s["k_pages"], s["k_scale"], ids, slots, s["k"], c["cache"])
    _put(s["v_pages"], s["v_scale"], ids, slots, s["v"], c["cache"])
    k = _gather(s["k_pages"], s["k_scale"], table)
    x = torch.matmul(q.float().view(B, c["Hkv"], c["G"], D), k.transpose(2, 3)) * D ** -0.5
    del k
    x = x.masked_fill(torch.arange(x.shape[-1], device=DEV) > pos[:, None, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    # Values at positions behind the last are no part of the sum, whatever the pages hold there.
    v = _gather(s["v_pages"], s["v_scale"], table)
    v = v.masked_fill((torch.arange(v.shape[2], device=DEV) > pos[:, None])[:, None, :, None], 0.0)
    return torch.matmul(x, v).view(B, H, D).to(q.dtype)


def _plain_write(s):
    c = s["case"]
    i = torch.arange(c["N"], device=DEV)
    b, i = torch.nonzero(i < s["counts"][:, None], as_tuple=True)
    at = s["pos"][b] + i
    ids, slots = s["page_table"][b, at // c["page"]].long(), at % c["page"]
    _put(s["k_pages"], s["k_scale"], ids, slots, s["k"][b, :, i], c["cache"])
    _put(s["v_pages"], s["v_scale"], ids, slots, s["v"][b, :, i], c["cache"])


def _plain_read(s):
    c = s["case"]
    past = (torch.arange(c["T"], device=DEV) >= s["lengths"][:, None])[:, None, :, None]
    return tuple(_gather(s[n + "_pages"], s[n + "_scale"], s["page_table"])[:, :, :c["T"]]
                 .masked_fill(past, 0.0).to(DTYPES[c["dtype"]]) for n in "kv")


def run(s):
    op, narrow = s["case"]["op"], s["k_scale"] is not None
    if op == "step":
        out = _own_step(s) if own else _plain_step(s)
        # The updated state: an 8-bit pool is its values up to the rows' scales, and those.
        return dict(out=out, k_pages=s["k_pages"], v_pages=s["v_pages"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if op == "write":
        _own_write(s) if own else _plain_write(s)
        if not narrow:
            return dict(k_pages=s["k_pages"], v_pages=s["v_pages"])
    k, v = _own_read(s) if own else _plain_read(s)
    return dict(k=k, v=v)


def work(c):
    n, e, z = sum(_lengths(c)), SIZES[c["dtype"]], SIZES[c["cache"]]
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    row = 2 * Hkv * (D * z + (z == 1))  # a position's key and value rows in the pools
    new = 2 * Hkv * D * e               # ... as the caller has them
    pages = 4 * sum(-(-x // c["page"]) for x in _lengths(c))
    if c["op"] == "step":
        heads = Hkv * c["G"] * D
        return dict(bytes=(n - B) * row + B * (new + row) + 2 * B * heads * e + pages + 8 * B, flops=4.0 * n * heads)
    b = 0
    if c["op"] == "write":
        b = sum(_counts(c)) * (new + row) + pages + 16 * B
    if c["op"] == "read" or z == 1:
        b += n * row + B * c["T"] * new + pages + 8 * B
    return dict(bytes=b, flops=0.0)


# ---- From the definition, in 64 bits. -----------------------------------------------------------

def _pow2(e):
    """2^e exactly, e whole numbers in float64."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored64(x, cache):
    """What an 8-bit cache keeps of the rows x (float64)."""
    top, bits = (448.0, 3) if cache == "e4m3" else (127.0, None)
    size = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(size / top)).clamp(min=-200.0)
    e = torch.where(size > top * _pow2(e), e + 1, torch.where(size <= top * _pow2(e - 1), e - 1, e))
    e = torch.where(size == 0, torch.full_like(e, -127.0), e.clamp(min=-127.0))
    y = x / _pow2(e)
    if bits is None:
        step = torch.ones_like(y)
    else:  # three bits behind the leading one, down to steps of 2^-9
        lead = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30)))
        lead = torch.where(y.abs() >= _pow2(lead + 1), lead + 1, torch.where(y.abs() < _pow2(lead), lead - 1, lead))
        step = _pow2(lead.clamp(min=-6.0) - bits)
    return torch.round(y / step) * step * _pow2(e)


def _stored_rows(s, n, b, length):
    """The rows 0 .. length - 1 of sequence b in pool n ("k" or "v"), [Hkv, length, D] float64."""
    page = s["case"]["page"]
    ids = s["page_table"][b, :-(-length // page)].tolist()
    rows = torch.cat([s[n + "_pages"][i].double() for i in ids], dim=1)
    if s[n + "_scale"] is not None:
        e = torch.cat([s[n + "_scale"][i].view(torch.uint8) for i in ids], dim=1).double()
        rows = rows * _pow2(e - 127.0)[..., None]
    return rows[:, :length].clone()


def exact(c, seed):
    s = prepare(c, seed)
    op, cache, dt = c["op"], c["cache"], DTYPES[c["dtype"]]
    if op == "write" and SIZES[cache] > 1:
        return None  # rows are copied: nothing is computed
    keep = (lambda x: _stored64(x, cache)) if SIZES[cache] == 1 else (lambda x: x)
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    if op == "step":
        out = torch.empty(B, Hkv, c["G"], D, dtype=torch.float64, device=DEV)
        for b, length in enumerate(_lengths(c)):
            k, v = (_stored_rows(s, n, b, length) for n in "kv")
            k[:, length - 1], v[:, length - 1] = keep(s["k"][b].double()), keep(s["v"][b].double())
            w = torch.softmax(s["q"][b].double().view(Hkv, c["G"], D) @ k.mT.contiguous() / math.sqrt(D), dim=-1)
            out[b] = w @ v
        return dict(out=out.view(B, Hkv * c["G"], D), k_pages=None, v_pages=None, k_scale=None, v_scale=None)
    res = {n: torch.zeros(B, Hkv, c["T"], D, dtype=torch.float64, device=DEV) for n in "kv"}
    for b, length in enumerate(_lengths(c)):
        for n in "kv":
            res[n][b, :, :length] = _stored_rows(s, n, b, length)
            if op == "write":
                m = _counts(c)[b]
                res[n][b, :, length - m:length] = keep(s[n][b, :, :m].double())
    return res
