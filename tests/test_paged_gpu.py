"""The paged key/value cache on the GPU against the 64-bit oracle: stored rows bit for bit, attention within a
bound that counts its roundings (oracle/paged_oracle.py), over types, head layouts, lengths, page orders,
strides and what may stand in places that belong to nobody."""

import math

import pytest
import torch

import dwarf_amd
from dwarf_amd import PagedKVCache, paged_decode_step, paged_kv_read, paged_kv_write
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
F32, BF, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


class Cache:
    """Pools full of rows, with a page table in an order of no rule: everything a call needs, on the GPU, and
    the pools' copies on the CPU.  Pages and table entries that belong to nobody hold junk."""

    def __init__(self, dev, B, H, D, page, M, dtype, kv=None, lengths=None, layout="heads", seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.dtype, self.kv = dev, dtype, kv or dtype
        self.P = B * M + spare
        rows = torch.randn(self.P, H, page, D, generator=g) * torch.exp(torch.randn(self.P, H, page, 1, generator=g))
        rows2 = torch.randn(self.P, H, page, D, generator=g)
        self.narrow = self.kv.itemsize == 1
        self.k, self.k_scale = self._pool(rows, layout)
        self.v, self.v_scale = self._pool(rows2, layout)
        order = torch.randperm(self.P, generator=g)[:B * M].to(torch.int32).view(B, M)
        self.lengths = lengths
        if lengths is not None:  # entries behind a sequence's last page are no pages
            for b, n in enumerate(lengths):
                order[b, -(-max(n, 0) // page):] = [-1, 2 ** 31 - 1, -2 ** 31, self.P][b % 4]
        self.table = order.to(dev)

    def _pool(self, rows, layout):
        if not self.narrow:
            x, s = rows.to(self.kv), None
        else:  # any codes and scales are a valid pool
            if self.kv == I8:
                x = (rows * 40).clamp(-127, 127).to(I8)
            else:
                x = (rows * 100).clamp(-448, 448).to(E4)
            s = (rows.abs().amax(-1).log2().round() + 120).clamp(0, 254).to(torch.uint8).view(torch.float8_e8m0fnu).to(self.dev)
        x = x.to(self.dev)
        if layout == "tokens":  # [P, page, H, D] memory
            x = x.view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(self.kv) if self.narrow \
                else x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
            if s is not None:
                s = s.view(torch.uint8).permute(0, 2, 1).contiguous().permute(0, 2, 1).view(torch.float8_e8m0fnu)
        elif layout == "wide":  # a layer's share of a wider buffer
            y = x.view(torch.uint8)
            big = torch.full((y.shape[0], 2, *y.shape[1:3], y.shape[3] + 32), 0x7f, dtype=torch.uint8, device=self.dev)
            big[:, 1, :, :, :y.shape[3]] = y
            x = big[:, 1, :, :, :y.shape[3]].view(self.kv)
        return x, s

    @property
    def state(self):
        return dict(k_scale=self.k_scale, v_scale=self.v_scale)

    def cpu(self, t):
        return t.view(torch.uint8).cpu().view(t.dtype) if t.dtype.itemsize == 1 else t.cpu()

    def rows(self, n, b, length):
        """Rows 0 .. length - 1 of sequence b as the pool n ("k" or "v") holds them now."""
        s = getattr(self, n + "_scale")
        return po.sequence(self.cpu(getattr(self, n).contiguous()), self.table.cpu(), b, length, None if s is None else self.cpu(s))


def bits(t):
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.dtype.itemsize]).cpu()


def same(a, b):
    a, b = bits(a), bits(b)
    assert a.shape == b.shape
    n = int((a != b).sum())
    assert n == 0, f"{n} of {a.numel()} elements differ, the first at {(a != b).nonzero()[0].tolist()}"


def junk(c, lengths):
    """NaN and infinities in every row of the pools that no sequence uses."""
    page = c.k.shape[2]
    used = torch.zeros(c.P, page, dtype=torch.bool)
    table = c.table.cpu()
    for b, n in enumerate(lengths):
        for t in range(max(0, n)):
            i = int(table[b, t // page]) if t // page < table.shape[1] else -1
            if 0 <= i < c.P:
                used[i, t % page] = True
    mask = (~used).to(c.dev)[:, None, :, None]
    for i, x in enumerate((c.k, c.v)):
        if c.narrow:
            x.view(torch.uint8).masked_fill_(mask, 0x7f if i == 0 else 0xff)
        else:
            x.masked_fill_(mask, math.inf if i == 0 else math.nan)
    for s in (c.k_scale, c.v_scale):
        if s is not None:
            s.view(torch.uint8).masked_fill_(mask[..., 0], 255)


# ---- Writing. -------------------------------------------------------------------------------------------

def _rows(dev, dtype, layout, B, H, N, D, seed=5):
    g = torch.Generator().manual_seed(seed)
    if layout == "qkv":         # head views of a projection output
        t = torch.randn(B, N, 3 * H * D, generator=g).to(dev, dtype)
        return [u.view(B, N, H, D).permute(0, 2, 1, 3) for u in t.split(H * D, dim=-1)[1:]]
    if layout == "expanded":    # one prompt for every sequence
        return [torch.randn(1, H, N, D, generator=g).to(dev, dtype).expand(B, H, N, D) for _ in range(2)]
    if layout == "unaligned":
        return [torch.randn(B, H, N, D + 1, generator=g).to(dev, dtype)[..., 1:] for _ in range(2)]
    if layout == "negated":
        return [torch._neg_view(torch.randn(B, H, N, D, generator=g).to(dev, dtype)) for _ in range(2)]
    return [torch.randn(B, H, N, D, generator=g).to(dev, dtype) for _ in range(2)]


def _expect_write(c, k, v, pos, counts):
    """The pools (and scales) on the CPU after a write."""
    page, table = c.k.shape[2], c.table.cpu()
    out = []
    for rows, pool, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        x, s = c.cpu(pool.contiguous()).clone(), None if scale is None else c.cpu(scale.contiguous()).view(torch.uint8).clone()
        rows = rows.cpu()
        for b in range(rows.shape[0]):
            for i in range(rows.shape[2] if counts is None else min(rows.shape[2], counts[b])):
                t = pos[b] + i
                if t < 0 or t // page >= table.shape[1] or not 0 <= int(table[b, t // page]) < c.P:
                    continue
                p = int(table[b, t // page])
                if scale is None:
                    x[p, :, t % page] = rows[b, :, i]
                else:
                    codes, e = po.encode(rows[b, :, i], c.kv)
                    x.view(torch.uint8)[p, :, t % page] = codes.float().to(c.kv).view(torch.uint8)
                    s[p, :, t % page] = e
        out += [x, s]
    return out


def _check_write(c, k, v, pos, counts):
    want = _expect_write(c, k, v, pos, counts)
    dev = c.dev
    version = c.k._version
    paged_kv_write(k, v, c.k, c.v, c.table, torch.tensor(pos, device=dev),
                   counts=None if counts is None else torch.tensor(counts, device=dev), **c.state)
    assert c.k._version > version
    for got, ref in zip((c.k, c.k_scale, c.v, c.v_scale), want):
        if ref is not None:
            same(got, ref)


@pytest.mark.parametrize("layout", ["plain", "qkv", "expanded", "unaligned", "negated"])
@pytest.mark.parametrize("dtype,kv", [(F32, None), (BF, None), (F16, None), (BF, E4), (BF, I8), (F16, E4), (F16, I8),
                                      (F32, E4), (F32, I8)])
def test_write_layouts_and_types(gpu_device, dtype, kv, layout):
    c = Cache(gpu_device, 2, 3, 64, 16, 3, dtype, kv)
    k, v = _rows(gpu_device, dtype, layout, 2, 3, 21, 64)
    _check_write(c, k, v, [0, 19], [21, 20])


@pytest.mark.parametrize("D", [32, 80, 96, 128])
@pytest.mark.parametrize("kv", [None, E4, I8])
@pytest.mark.parametrize("pool", ["heads", "tokens", "wide"])
def test_write_head_dims_and_pools(gpu_device, D, kv, pool):
    c = Cache(gpu_device, 2, 2, D, 32, 2, BF, kv, layout=pool)
    k, v = _rows(gpu_device, BF, "plain", 2, 2, 33, D)
    _check_write(c, k, v, [31, 5], None)


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 150])
def test_write_lengths(gpu_device, N):
    """Rows that end inside a page, reach past the table, start before it, or are none."""
    c = Cache(gpu_device, 5, 2, 32, 16, 6, BF, lengths=[96, 40, 96, 96, 17])
    k, v = _rows(gpu_device, BF, "plain", 5, 2, N, 32)
    _check_write(c, k, v, [0, 15, 95, -3, 10], [N, N + 7, N, N, -1 if N == 2 else N // 2])


def test_write_far_positions_and_bad_pages(gpu_device):
    c = Cache(gpu_device, 6, 2, 32, 16, 4, BF, I8)
    c.table[1, 1], c.table[2, 1], c.table[3, 0] = -1, c.P, 2 ** 31 - 1
    k, v = _rows(gpu_device, BF, "plain", 6, 2, 40, 32)
    _check_write(c, k, v, [0, 3, 3, 3, 2 ** 40, -2 ** 62], None)


def _edge_rows(dtype, D):
    """Rows where a scale or a rounding can go wrong."""
    fi = torch.finfo(dtype)
    tiny = fi.smallest_normal * fi.eps
    g = torch.Generator().manual_seed(9)
    r = torch.randn(64, D, generator=g).double()
    rows = [torch.zeros(D), -torch.zeros(D)]
    for top in (448.0, 127.0):
        for f in (1.0, 1 + fi.eps, 1 - fi.eps / 2, 2.0, 0.5):
            x = r[0].clone() * 0.01
            x[3] = top * f
            rows.append(x)
    rows.append(torch.arange(D) + 0.5)                      # halves of an integer's step
    rows.append((torch.arange(D) + 0.5) / 127 * 127)
    rows.append(torch.cat([torch.tensor([448.0, 17.0, 19.0, 21.0, 23.0, 2 ** -9, 2 ** -10, 3 * 2 ** -10]), torch.zeros(D - 8)]))
    rows += [torch.full((D,), tiny), torch.full((D,), -tiny), r[1] * fi.smallest_normal, r[2] * tiny * 9]
    rows += [torch.full((D,), fi.max), -torch.full((D,), fi.max), r[3] * fi.max / 5]
    for bad in (math.inf, -math.inf, math.nan):
        x = r[4].clone()
        x[D - 1] = bad
        rows.append(x)
    x = r[5].clone()
    x[0], x[1] = math.nan, math.inf
    rows.append(x)
    rows += list(r[6:] * torch.exp(4 * torch.randn(58, 1, generator=g)))
    return torch.stack([x.double() for x in rows]).to(dtype)


@pytest.mark.parametrize("D", [32, 64, 80])
@pytest.mark.parametrize("kv", [E4, I8])
@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_write_and_read_rows_at_the_edges(gpu_device, dtype, kv, D):
    """Stored and read back, through the write and through the decode step, bit for bit."""
    x = _edge_rows(dtype, D)
    n = x.shape[0]
    rows = x.to(gpu_device)[None, None]
    c = Cache(gpu_device, 1, 1, D, 16, -(-n // 16), dtype, kv)
    _check_write(c, rows, rows.flip(-1), [0], None)
    codes, e = po.encode(x, kv)
    val = codes * torch.where(e == 255, torch.tensor(math.nan, dtype=torch.float64), 2.0 ** (e.double() - 127))[:, None]
    length = torch.tensor([n], device=gpu_device)
    for out in (F32, BF, F16):
        k, v = paged_kv_read(c.k, c.v, c.table, length, n, dtype=out, **c.state)
        # (float64 -> float32 is exact here: 8 bits times a power of two in float32's range or below it,
        # where both sides round alike.)
        want = val.float().to(out)
        assert torch.equal(torch.isnan(k[0, 0].cpu()), torch.isnan(want))
        assert torch.equal(k[0, 0].cpu().nan_to_num(0.5), want.nan_to_num(0.5))
        assert torch.equal(v[0, 0].flip(-1).cpu().nan_to_num(0.5), want.nan_to_num(0.5))
    d = Cache(gpu_device, n, 1, D, 16, 1, dtype, kv)
    want = _expect_write(d, rows[0, 0][:, None, None], rows[0, 0][:, None, None], [3] * n, None)
    r = rows[0, 0][:, None]
    paged_decode_step(r, r, r, d.k, d.v, d.table, torch.full((n,), 3, device=gpu_device), **d.state)
    for got, ref in zip((d.k, d.k_scale, d.v, d.v_scale), want):
        same(got, ref)


def test_every_16_bit_value_rounds_as_torch_does(gpu_device):
    """e4m3 codes of all bfloat16 values up to 448 under a scale of one."""
    x = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(BF).float()
    x = x[x.abs() <= 448].to(BF)
    x = torch.cat([x, torch.zeros(-len(x) % 31, dtype=BF)]).view(-1, 31)
    x = torch.cat([torch.full((len(x), 1), 448.0, dtype=BF), x], 1)
    n = len(x)
    c = Cache(gpu_device, 1, 1, 32, 64, -(-n // 64), BF, E4)
    rows = x.to(gpu_device)[None, None]
    paged_kv_write(rows, rows, c.k, c.v, c.table, torch.zeros(1, dtype=torch.int64, device=gpu_device), **c.state)
    k, _ = paged_kv_read(c.k, c.v, c.table, torch.tensor([n], device=gpu_device), n, dtype=F32, **c.state)
    assert torch.equal(k[0, 0].cpu(), x.to(E4).float())


# ---- Reading. ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("out", [F32, BF, F16])
@pytest.mark.parametrize("kv", [F32, BF, F16, E4, I8])
def test_read_types(gpu_device, kv, out):
    lengths = [50, 0, 33, 1]
    dtype = kv if kv.itemsize > 1 else out
    c = Cache(gpu_device, 4, 3, 64, 16, 4, dtype, kv, lengths)
    junk(c, lengths)
    k, v = paged_kv_read(c.k, c.v, c.table, torch.tensor(lengths, device=gpu_device), 57, dtype=out, **c.state)
    for b, n in enumerate(lengths):
        for name, x in (("k", k), ("v", v)):
            want = c.rows(name, b, n).float().to(out)
            assert torch.equal(x[b, :, :n].cpu(), want)
            assert (x[b, :, n:] == 0).all()
    assert k.dtype == out and k.shape == (4, 3, 57, 64)


@pytest.mark.parametrize("D", [32, 80, 96, 128])
@pytest.mark.parametrize("pool", ["heads", "tokens", "wide"])
@pytest.mark.parametrize("kv", [BF, I8])
def test_read_head_dims_and_pools(gpu_device, D, pool, kv):
    lengths = [17, 64]
    c = Cache(gpu_device, 2, 2, D, 32, 2, BF, kv, lengths, layout=pool)
    k, v = paged_kv_read(c.k, c.v, c.table, torch.tensor(lengths, dtype=torch.int32, device=gpu_device), **c.state)
    assert k.shape == (2, 2, 64, D) and k.dtype == BF
    for b, n in enumerate(lengths):
        assert torch.equal(k[b, :, :n].cpu(), c.rows("k", b, n).float().to(BF))
        assert torch.equal(v[b, :, :n].cpu(), c.rows("v", b, n).float().to(BF))


def test_read_past_the_table_and_bad_pages(gpu_device):
    c = Cache(gpu_device, 3, 2, 32, 16, 2, BF)
    c.table[1, 0], c.table[2, 1] = -1, c.P
    k, v = paged_kv_read(c.k, c.v, c.table, torch.tensor([40, 20, 2 ** 40], device=gpu_device), 45)
    for x in (k, v):
        nan = torch.isnan(x).all(1).all(-1).cpu()
        want = torch.zeros(3, 45, dtype=torch.bool)
        want[0, 32:40] = want[1, :16] = want[2, 16:] = True
        assert torch.equal(nan, want) and not torch.isnan(x.cpu()[~want[:, None].expand(3, 2, 45)]).any()
        assert (x[0, :, 40:] == 0).all() and (x[1, :, 20:] == 0).all()


# ---- The decode step. --------------------------------------------------------------------------------------

def _step(c, pos, G=1, fresh=True, scale=None, seed=3, q=None):
    """Runs a step and checks its output and the rows that it wrote against the oracle."""
    B, (P, H, page, D), dev = len(pos), c.k.shape, c.dev
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, H * G, D, generator=g) * 2).to(dev, c.dtype) if q is None else q
    kn, vn = (torch.randn(B, H, D, generator=g).to(dev, c.dtype) for _ in range(2)) if fresh else (None, None)
    if fresh:
        want = _expect_write(c, kn[:, :, None], vn[:, :, None], pos, None)
    else:
        want = [None if t is None else c.cpu(t.contiguous()).clone() for t in (c.k, c.k_scale, c.v, c.v_scale)]
    out = paged_decode_step(q, kn, vn, c.k, c.v, c.table, torch.tensor(pos, device=dev), softmax_scale=scale, **c.state)
    for got, ref in zip((c.k, c.k_scale, c.v, c.v_scale), want):
        if ref is not None:
            same(got, ref)
    assert out.dtype == c.dtype and out.shape == q.shape
    worst = 0.0
    for b, p in enumerate(pos):
        x = out[b].double().cpu()
        if p < 0:
            assert (x == 0).all()
            continue
        if p >= c.table.shape[1] * page:
            assert torch.isnan(x).all()
            continue
        k, v = c.rows("k", b, p + 1), c.rows("v", b, p + 1)
        if torch.isnan(k).any() or torch.isnan(v).any():
            assert torch.isnan(x).all()
            continue
        ref, mass, size = po.attend(q[b].cpu(), k, v, D ** -0.5 if scale is None else scale)
        tol = po.bound(ref, mass, size, D, p + 1, c.dtype)
        ratio = ((x - ref).abs() / tol).max().item()
        assert ratio <= 1, f"sequence {b}: {ratio:.3g} of the bound"
        worst = max(worst, ratio)
    return out


@pytest.mark.parametrize("D", [32, 64, 80, 96, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 7, 8, 17])
@pytest.mark.parametrize("dtype,kv", [(F32, None), (BF, None), (F16, None), (BF, E4), (F16, I8), (F32, E4), (BF, I8), (F16, E4),
                                      (F32, I8)])
def test_step_types_and_heads(gpu_device, dtype, kv, G, D):
    pos = [299, 0, 130, 63]
    c = Cache(gpu_device, 4, 2, D, 32, 10, dtype, kv, [p + 1 for p in pos])
    junk(c, [p + 1 for p in pos])
    _step(c, pos, G)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("dtype,kv,G", [(BF, None, 1), (F32, None, 2), (BF, E4, 4), (F16, None, 8), (F16, I8, 5)])
def test_step_lengths(gpu_device, dtype, kv, G, page):
    """Lengths around the tiles, the chunks and the pages, with and without a new row."""
    pos = [0, 1, 2, 14, 15, 16, 17, 31, 62, 63, 64, 65, 127, 128, 129, 130, 255, 256, 257, 511, 512, 513, 640, 1023, -1]
    M = -(-1024 // page)
    c = Cache(gpu_device, len(pos), 1, 64, page, M, dtype, kv, [p + 1 for p in pos])
    junk(c, [p + 1 for p in pos])
    for fresh in (True, False):
        _step(c, pos, G, fresh)


@pytest.mark.parametrize("dtype,kv,G,D", [(BF, None, 1, 64), (F32, None, 1, 32), (BF, E4, 4, 128), (F16, I8, 6, 80)])
def test_step_long_sequences(gpu_device, dtype, kv, G, D):
    pos = [20000, 9999, 0]
    c = Cache(gpu_device, 3, 1, D, 128, 160, dtype, kv, [p + 1 for p in pos])
    junk(c, [p + 1 for p in pos])
    a = _step(c, pos, G)
    b = _step(c, pos, G)
    assert torch.equal(a, b)


@pytest.mark.parametrize("D", [32, 64, 80, 96, 128])
@pytest.mark.parametrize("dtype,kv,G", [(F32, None, 1), (BF, None, 3), (F16, None, 17), (BF, E4, 8), (F16, I8, 5), (F32, E4, 4),
                                        (F32, I8, 2)])
def test_step_joins(gpu_device, dtype, kv, G, D):
    """Sequences of one part to a dozen, whose last parts have a row or are full."""
    pos = [1500, 127, 128, 129, 640, 383, 0, -1, 896]
    c = Cache(gpu_device, len(pos), 2, D, 32, 48, dtype, kv, [p + 1 for p in pos])
    junk(c, [p + 1 for p in pos])
    for fresh in (True, False):
        _step(c, pos, G, fresh)


@pytest.mark.parametrize("B,H,dtype,kv,D,G", [(64, 4, BF, None, 64, 2), (32, 16, BF, E4, 128, 4), (47, 11, F32, None, 32, 1),
                                              (26, 20, F16, I8, 80, 5)])
def test_step_many_units(gpu_device, B, H, dtype, kv, D, G):
    """Heads and sequences enough that a workgroup takes all rows of one."""
    g = torch.Generator().manual_seed(B)
    pos = (torch.rand(B, generator=g) ** 2 * 1023).long().tolist()
    pos[0], pos[1], pos[2], pos[3] = 1023, -1, 0, 1024
    c = Cache(gpu_device, B, H, D, 64, 16, dtype, kv, [min(p, 1023) + 1 for p in pos])
    junk(c, [p + 1 for p in pos])
    _step(c, pos, G)


class RaggedCache(Cache):
    """A pool of just the pages that the lengths need, under a table for sequences of up to M pages."""

    def __init__(self, dev, H, D, page, M, dtype, kv, lengths, seed=0):
        used = [-(-max(n, 0) // page) for n in lengths]
        super().__init__(dev, 1, H, D, page, sum(used), dtype, kv, seed=seed)
        order, table, at = self.table[0].cpu(), torch.full((len(lengths), M), -1, dtype=torch.int32), 0
        for b, u in enumerate(used):
            table[b, :u] = order[at:at + u]
            at += u
        self.table, self.lengths = table.to(dev), lengths


@pytest.mark.parametrize("B,H,G,D,dtype,kv,most", [
    (40, 4, 1, 64, BF, None, 2200), (40, 4, 3, 64, F16, None, 2200), (40, 4, 2, 128, BF, None, 1300), (33, 4, 4, 96, BF, E4, 1500),
    (300, 1, 20, 32, BF, I8, 700), (512, 1, 2, 32, F16, E4, 400), (7, 20, 1, 80, BF, None, 3000)])
def test_step_shares(gpu_device, B, H, G, D, dtype, kv, most):
    """Large batches under long tables, whose rows the kernel deals out in equal shares: shares of several
    sequences, sequences of several shares, rows that end anywhere, sequences without rows."""
    g = torch.Generator().manual_seed(B)
    pos = (torch.rand(B, generator=g) ** 2 * most).long().tolist()
    pos[0], pos[1], pos[2], pos[-1], pos[-2] = 127, 128, -1, 255, 256
    M = 16 * 768 * 16 * 128 // (B * H * 32) + 64
    c = RaggedCache(gpu_device, H, D, 32, M * 2, dtype, kv, [p + 1 for p in pos])
    junk(c, [p + 1 for p in pos])
    pos[3] = c.table.shape[1] * 32 + 5  # past the table
    for fresh in (True, False):
        a = _step(c, pos, G, fresh)
    same(_step(c, pos, G, False), a)


@pytest.mark.parametrize("pool", ["tokens", "wide"])
@pytest.mark.parametrize("dtype,kv,G", [(BF, None, 1), (F32, None, 2), (BF, E4, 4), (F16, I8, 8), (BF, None, 8)])
def test_step_pools(gpu_device, dtype, kv, G, pool):
    pos = [200, 77, 16]
    _step(Cache(gpu_device, 3, 3, 64, 16, 13, dtype, kv, [p + 1 for p in pos], layout=pool), pos, G)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 3.0])
@pytest.mark.parametrize("G", [1, 4])
def test_step_softmax_scale(gpu_device, scale, G):
    """A flat softmax, a sharp one and a reversed one."""
    pos = [300, 45]
    _step(Cache(gpu_device, 2, 2, 64, 64, 5, F32, None, [p + 1 for p in pos]), pos, G, scale=scale)


@pytest.mark.parametrize("G", [1, 2, 8])
@pytest.mark.parametrize("kv", [None, I8])
def test_step_bad_pages_and_positions(gpu_device, kv, G):
    """A sequence that attends a position without a page gets NaN, and no other one does."""
    pos = [40, 40, 40, 40, 64, 2 ** 33 + 5, -1, -2 ** 40, 30]
    c = Cache(gpu_device, len(pos), 2, 32, 16, 4, BF, kv)
    c.table[0, 0], c.table[1, 2], c.table[2, 1], c.table[8, 3] = -1, c.P, -2 ** 31, -7
    out = _step(c, pos, G)
    nan = torch.isnan(out).all(-1).all(-1).tolist()
    assert nan == [True, True, True, False, True, True, False, False, False]
    out = _step(c, pos, G, fresh=False)
    assert torch.isnan(out).all(-1).all(-1).tolist() == nan


@pytest.mark.parametrize("dtype,kv,G", [(BF, None, 1), (BF, None, 4), (F32, None, 1), (BF, E4, 8), (F16, None, 4)])
def test_step_special_values(gpu_device, dtype, kv, G):
    """NaN and infinities in a sequence's own rows make that sequence's heads what the formula makes them."""
    pos = [150] * 6
    c = Cache(gpu_device, 6, 2, 64, 16, 10, dtype, kv, [p + 1 for p in pos])
    page = lambda b, t: int(c.table[b, t // 16])
    if kv is None:
        c.k[page(0, 70), 0, 70 % 16, 5] = math.nan
        c.v[page(1, 3), 1, 3, 9] = math.nan
        c.v[page(2, 149), 0, 149 % 16, 9] = math.inf
        c.k[page(3, 20), 1, 20 % 16] = math.inf
    else:
        c.k_scale.view(torch.uint8)[page(0, 70), 0, 70 % 16] = 255
        c.v_scale.view(torch.uint8)[page(1, 3), 1, 3] = 255
        c.v_scale.view(torch.uint8)[page(2, 149), 0, 149 % 16] = 255
        c.k_scale.view(torch.uint8)[page(3, 20), 1, 20 % 16] = 255
    q = torch.ones(6, 2 * G, 64, device=gpu_device, dtype=dtype)
    out = paged_decode_step(q, None, None, c.k, c.v, c.table, torch.tensor(pos, device=gpu_device), **c.state).float().cpu()
    nan = torch.isnan(out.view(6, 2, G, 64))
    assert nan[0, 0].all() and not nan[0, 1].any()
    assert nan[1, 1, :, 9 if kv is None else slice(None)].all() and not nan[1, 0].any()
    if kv is None:
        assert (out.view(6, 2, G, 64)[2, 0, :, 9] == math.inf).all() and nan[2].sum() == 0 and nan[1].sum() == G
    else:
        assert nan[2, 0].all() and not nan[2, 1].any()
    assert nan[3, 1].all() and not nan[3, 0].any()  # a score of +inf: inf - inf
    assert not nan[4:].any()


@pytest.mark.parametrize("dtype,kv,G", [(BF, None, 1), (BF, None, 8), (F16, None, 4), (F32, None, 1), (F32, None, 4)])
def test_step_ignores_values_of_no_weight(gpu_device, dtype, kv, G):
    """Values at the type's limits count for nothing where their weight is zero, in front of the row that has
    it all, behind it, and in the same tile."""
    n, D = 400, 64
    c = Cache(gpu_device, 1, 1, D, 16, 25, dtype, kv)
    table = c.table.cpu()[0]
    c.k.zero_()
    c.v.fill_(torch.finfo(dtype).max)
    c.k[int(table[200 // 16]), 0, 200 % 16] = 100.0
    c.v[int(table[200 // 16]), 0, 200 % 16] = torch.arange(D, device=gpu_device).to(dtype)
    q = torch.ones(1, G, D, device=gpu_device, dtype=dtype)  # a score of 800 against zeros
    out = paged_decode_step(q, None, None, c.k, c.v, c.table, torch.tensor([n - 1], device=gpu_device))
    assert torch.equal(out[0].float().cpu(), torch.arange(D).float().expand(G, D))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("kv", [E4, I8])
def test_every_code_reads_alike(gpu_device, kv, G, dtype):
    """All 256 codes under scales from the smallest to ones that overflow: what is read back, and the output of
    a step over one row, which is its value."""
    bytes_ = [0, 1, 60, 120, 127, 130, 200, 247, 254, 255]
    n = 8 * len(bytes_)
    c = Cache(gpu_device, n, 1, 32, 16, 1, dtype, kv)
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(8, 32).repeat(len(bytes_), 1)
    e = torch.tensor(bytes_, dtype=torch.uint8).repeat_interleave(8)
    page = c.table[:, 0].long()
    c.v.view(torch.uint8)[page, 0, 0] = codes.to(gpu_device)
    c.v_scale.view(torch.uint8)[page, 0, 0] = e.to(gpu_device)
    c.k.view(torch.uint8)[page, 0, 0] = 0
    want = po.values(codes.view(kv), e.view(torch.float8_e8m0fnu)).float().to(dtype)
    _, v = paged_kv_read(c.k, c.v, c.table, torch.ones(n, dtype=torch.int64, device=gpu_device), 1, dtype=dtype, **c.state)
    q = torch.ones(n, G, 32, device=gpu_device, dtype=dtype)
    out = paged_decode_step(q, None, None, c.k, c.v, c.table, torch.zeros(n, dtype=torch.int64, device=gpu_device), **c.state)
    for x in (v[:, 0, 0].cpu(), *out.unbind(1)):
        x = x.cpu()
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(x), nan)
        ok = ~nan
        # (The one weight is 2^-30 until the last division, in two terms of 8 bits: values below 2^-90 come near
        # the numbers that float32 holds to fewer bits, and the step promises them to 2^-94 only.)
        ok &= (want.float().abs() > 2.0 ** -90) | (want == 0)
        assert torch.equal(x[ok], want[ok])


def test_refuses_what_is_more_than_values(gpu_device):
    """Tangents, vmap's wrappers and gradients on a pool."""
    import torch.autograd.forward_ad as fw
    c = Cache(gpu_device, 1, 1, 32, 16, 1, BF)
    row, pos = torch.zeros(1, 1, 32, device=gpu_device, dtype=BF), torch.zeros(1, dtype=torch.int64, device=gpu_device)
    with fw.dual_level():
        for i in range(3):
            ops = [row, row.clone(), row.clone()]
            ops[i] = fw.make_dual(ops[i], ops[i].clone())
            with pytest.raises(RuntimeError):
                paged_decode_step(*ops, c.k, c.v, c.table, pos)
        with pytest.raises(RuntimeError):
            paged_kv_write(fw.make_dual(row[:, :, None], row[:, :, None].clone()), row[:, :, None], c.k, c.v, c.table, pos)
    before = c.k.clone()
    with pytest.raises(Exception):
        torch.vmap(lambda q: paged_decode_step(q, q, q, c.k, c.v, c.table, pos))(row[None])
    same(c.k, before)


@pytest.mark.parametrize("form", ["strided", "unaligned", "negated", "expanded"])
def test_step_operand_layouts(gpu_device, form):
    B, H, G, D = 3, 2, 4, 64
    g = torch.Generator().manual_seed(8)
    if form == "strided":    # one token's projection output
        t = torch.randn(B, (H * G + 2 * H) * D, generator=g).to(gpu_device, BF)
        q, k, v = t.split([H * G * D, H * D, H * D], dim=1)
        q, k, v = q.view(B, H * G, D), k.view(B, H, D), v.view(B, H, D)
    elif form == "unaligned":
        q, k, v = (torch.randn(B, h, D + 1, generator=g).to(gpu_device, BF)[..., 1:] for h in (H * G, H, H))
    elif form == "negated":
        q, k, v = (torch._neg_view(torch.randn(B, h, D, generator=g).to(gpu_device, BF)) for h in (H * G, H, H))
    else:
        q, k, v = (torch.randn(1, 1, D, generator=g).to(gpu_device, BF).expand(B, h, D) for h in (H * G, H, H))
    pos = torch.tensor([100, 30, 0], dtype=torch.int32, device=gpu_device)
    res = []
    for ops in ((q, k, v), [t.resolve_neg().contiguous() for t in (q, k, v)]):
        c = Cache(gpu_device, B, H, D, 16, 7, BF)
        wide = torch.stack([c.table, c.table + 1], 2)[:, :, 0]  # a table with strides
        res.append((paged_decode_step(*ops, c.k, c.v, wide, pos), c.k, c.v))
    for a, b in zip(*res):
        same(a, b)


def test_step_shares_pages(gpu_device):
    """Sequences with a common prefix read the same pages; the copies' results are theirs."""
    c = Cache(gpu_device, 4, 2, 64, 16, 6, BF)
    c.table[1:, :4] = c.table[:1, :4]
    _step(c, [80, 80, 64, 95], 2)


def test_empty_calls(gpu_device):
    for B, H, M in ((0, 2, 3), (2, 0, 3), (2, 2, 0)):
        c = Cache(gpu_device, B, H, 32, 16, M, BF)
        pos = torch.zeros(B, dtype=torch.int64, device=gpu_device)
        row = torch.zeros(B, H, 32, device=gpu_device, dtype=BF)
        out = paged_decode_step(row, row, row, c.k, c.v, c.table, pos)
        assert out.shape == (B, H, 32) and torch.isnan(out).all()
        paged_kv_write(row[:, :, None], row[:, :, None], c.k, c.v, c.table, pos)
        k, _ = paged_kv_read(c.k, c.v, c.table, pos, 5)
        assert k.shape == (B, H, 5, 32) and (k == 0).all()
    c = Cache(gpu_device, 2, 2, 32, 16, 3, BF)
    none = torch.zeros(2, 2, 0, 32, device=gpu_device, dtype=BF)
    paged_kv_write(none, none, c.k, c.v, c.table, torch.zeros(2, dtype=torch.int64, device=gpu_device))
    assert paged_kv_read(c.k, c.v, c.table, torch.ones(2, dtype=torch.int64, device=gpu_device), 0)[0].shape == (2, 2, 0, 32)


@pytest.mark.parametrize("kv", [BF, I8])
def test_pools_past_32_bits(gpu_device, kv):
    """Rows whose byte offsets need more than 32 bits."""
    D, page, H = 128, 256, 8
    P = (5 << 30) // (H * page * D * kv.itemsize)
    k, v = (torch.empty(P, H, page, D, device=gpu_device, dtype=kv) for _ in range(2))
    scale = {}
    if kv == I8:
        scale = {n: torch.empty(P, H, page, device=gpu_device, dtype=torch.uint8).view(torch.float8_e8m0fnu)
                 for n in ("k_scale", "v_scale")}
    table = torch.tensor([[P - 1, 0, P // 2], [1, P - 2, P - 3]], dtype=torch.int32, device=gpu_device)
    g = torch.Generator().manual_seed(4)
    N = 600
    rows = [torch.randn(2, H, N, D, generator=g).to(BF) for _ in range(2)]
    pos = torch.zeros(2, dtype=torch.int64, device=gpu_device)
    paged_kv_write(*(r.to(gpu_device) for r in rows), k, v, table, pos, **scale)
    got = paged_kv_read(k, v, table, pos + N, N, dtype=F32, **scale)
    q = torch.randn(2, H, D, generator=g).to(BF)
    out = paged_decode_step(q.to(gpu_device), None, None, k, v, table, pos + N - 1, **scale).cpu().double()
    for x, r in zip(got, rows):
        if kv == BF:
            assert torch.equal(x.cpu(), r.float())
        else:  # half a step of a scale that is at most 2 amax / 127
            assert ((x.cpu() - r.float()).abs() <= r.float().abs().amax(-1, keepdim=True) / 127).all()
    for b in range(2):
        ref, mass, size = po.attend(q[b], got[0][b].cpu().double(), got[1][b].cpu().double(), D ** -0.5)
        assert ((out[b] - ref).abs() <= po.bound(ref, mass, size, D, N, BF)).all()


# ---- Streams, graphs, devices' rules. -----------------------------------------------------------------------

@pytest.mark.parametrize("kv", [None, E4])
def test_other_streams(gpu_device, kv):
    """Calls on a stream of their own, with another one at work between, give what they give alone."""
    mk = lambda: Cache(gpu_device, 2, 2, 64, 16, 40, BF, kv, seed=7)
    a, b = mk(), mk()
    ra, rb = mk(), mk()
    pos = torch.tensor([600, 299], device=gpu_device)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, h, 64, generator=g).to(gpu_device, BF) for h in (8, 2, 2))
    want = [paged_decode_step(q, k, v, c.k, c.v, c.table, pos, **c.state) for c in (ra, rb)]
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        for c, stream in ((a, s), (b, t)):
            with torch.cuda.stream(stream):
                got.append(paged_decode_step(q, k, v, c.k, c.v, c.table, pos, **c.state))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2])
    same(a.k, ra.k)
    same(b.v, rb.v)


@pytest.mark.parametrize("kv,G", [(None, 1), (I8, 4)])
def test_graphs(gpu_device, kv, G):
    """Two captured steps, of two caches, replayed in turn with eager work between them: each replay writes
    the row at the position that it finds and gives the eager result."""
    mk = lambda s: Cache(gpu_device, 2, 2, 64, 16, 60, BF, kv, seed=s)
    caches, refs = [mk(1), mk(2)], [mk(1), mk(2)]
    starts = [[500, 3], [30, 900]]
    g = torch.Generator().manual_seed(1)
    rows = [[torch.randn(2, h, 64, generator=g).to(gpu_device, BF) for h in (2 * G, 2, 2)] for _ in range(6)]
    want = []
    for c, start in zip(refs, starts):
        p = torch.tensor(start, device=gpu_device)
        want.append([])
        for r in rows:
            want[-1].append(paged_decode_step(*r, c.k, c.v, c.table, p, **c.state))
            p += 1
    ins = [[t.clone() for t in rows[0]] for _ in range(2)]
    pos = [torch.tensor(s, device=gpu_device) for s in starts]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for c in (mk(3), mk(4)):  # warm-up, on caches of its own
            paged_decode_step(*rows[0], c.k, c.v, c.table, pos[0].clone(), **c.state)
    torch.cuda.synchronize()
    for c, i, p in zip(caches, ins, pos):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs.append(paged_decode_step(*i, c.k, c.v, c.table, p, **c.state))
            p += 1
        graphs.append(gr)
    for n, r in enumerate(rows):
        for w in range(2):
            for dst, src in zip(ins[w], r):
                dst.copy_(src)
            graphs[w].replay()
            eager = mk(5)
            paged_decode_step(*r, eager.k, eager.v, eager.table, torch.tensor([7, 8], device=gpu_device), **eager.state)
            torch.cuda.synchronize()
            assert torch.equal(outs[w], want[w][n]), (n, w)
    for c, r in zip(caches, refs):
        for x, y in ((c.k, r.k), (c.v, r.v)):
            same(x, y)


def test_refuses_mixed_devices_and_inference_tensors(gpu_device):
    c = Cache(gpu_device, 1, 1, 32, 16, 1, BF)
    row, pos = torch.zeros(1, 1, 32, device=gpu_device, dtype=BF), torch.zeros(1, dtype=torch.int64, device=gpu_device)
    for bad in (dict(pos=pos.cpu()), dict(q=row.cpu()), dict(page_table=c.table.cpu()), dict(v_new=row.cpu())):
        args = {**dict(q=row, k_new=row, v_new=row, k_pages=c.k, v_pages=c.v, page_table=c.table, pos=pos), **bad}
        with pytest.raises(RuntimeError, match="GPU|different devices"):
            paged_decode_step(**args)
    for bad in (dict(pos=pos.float()), dict(pos=pos[None]), dict(pos=torch.zeros(2, dtype=torch.int64, device=gpu_device))):
        args = {**dict(q=row, k_new=row, v_new=row, k_pages=c.k, v_pages=c.v, page_table=c.table, pos=pos), **bad}
        with pytest.raises(AssertionError, match="pos must be"):
            paged_decode_step(**args)
    for pages in (torch.zeros(1, 1, 16, 33, device=gpu_device, dtype=BF)[..., 1:],
                  torch.zeros(1, 1, 32, 16, device=gpu_device, dtype=BF).transpose(2, 3)):
        with pytest.raises(AssertionError, match="aligned"):
            paged_decode_step(row, row, row, pages, pages, c.table, pos)
    with pytest.raises(dwarf_amd._lib.DSQGLibraryError):  # rows that overlap
        e = torch.zeros(1, 1, 16, 32, device=gpu_device, dtype=BF).expand(4, 1, 16, 32)
        paged_decode_step(row, row, row, e, e, c.table, pos)
    with pytest.raises(dwarf_amd._lib.DSQGLibraryError):  # a head dim without kernels
        e, r = torch.zeros(1, 1, 16, 48, device=gpu_device, dtype=BF), torch.zeros(1, 1, 48, device=gpu_device, dtype=BF)
        paged_decode_step(r, r, r, e, e, c.table, pos)
    with torch.inference_mode():
        k, v = c.k.clone(), c.v.clone()
        paged_decode_step(row, row, row, k, v, c.table, pos)
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        paged_decode_step(row, row, row, k, v, c.table, pos)
    paged_decode_step(row, None, None, k, v, c.table, pos)  # (nothing is written)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_decode_step(row.clone().requires_grad_(), row, row, c.k, c.v, c.table, pos)
    with torch.no_grad():
        paged_decode_step(row.clone().requires_grad_(), row, row, c.k, c.v, c.table, pos)


def test_custom_ops_are_the_eager_calls(gpu_device):
    """What torch.compile traces: the same results as the eager functions."""
    def run(q, k, v, c, pos):
        out = paged_decode_step(q, k, v, c.k, c.v, c.table, pos, **c.state)
        paged_kv_write(k[:, :, None], v[:, :, None], c.k, c.v, c.table, pos + 1, **c.state)
        return (out, *paged_kv_read(c.k, c.v, c.table, pos + 2, 40, dtype=F32, **c.state))

    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, h, 32, generator=g).to(gpu_device, BF) for h in (6, 3, 3))
    pos = torch.tensor([20, 37], device=gpu_device)
    for kv in (None, I8):
        a, b = (Cache(gpu_device, 2, 3, 32, 16, 3, BF, kv) for _ in range(2))
        want = run(q, k, v, a, pos)
        with torch.no_grad():
            got = torch.compile(run, backend="aot_eager", fullgraph=True)(q, k, v, b, pos)
        for x, y in zip((*want, a.k, a.v), (*got, b.k, b.v)):
            same(x, y)


# ---- Together, as they are used. -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,kv", [(BF, None), (F32, None), (F16, None), (BF, E4), (F16, I8)])
def test_prompts_steps_and_reading_back(gpu_device, dtype, kv):
    """Ragged prompts, more rows, then steps: every step is attention over all rows so far, as they are read
    back."""
    B, H, G, D, counts = 3, 2, 2, 64, [70, 1, 33]
    g = torch.Generator().manual_seed(6)
    c = PagedKVCache(B, H, D, 100, dtype, gpu_device, kv_dtype=kv, page_size=16)
    k, v = (torch.randn(B, H, 70, D, generator=g).to(gpu_device, dtype) for _ in range(2))
    c.prefill(k, v, torch.tensor(counts, device=gpu_device))
    assert c.pos.tolist() == counts
    c.write(k[:, :, :5], v[:, :, :5])
    n = [x + 5 for x in counts]
    assert c.pos.tolist() == n
    for _ in range(6):
        q, kt, vt = (torch.randn(B, h, D, generator=g).to(gpu_device, dtype) for h in (H * G, H, H))
        out = c.step(q, kt, vt).double().cpu()
        n = [x + 1 for x in n]
        assert c.pos.tolist() == n
        rk, rv = c.read(dtype=F32)
        for b in range(B):
            ref, mass, size = po.attend(q[b].cpu(), rk[b, :, :n[b]].cpu().double(), rv[b, :, :n[b]].cpu().double(), D ** -0.5)
            assert ((out[b] - ref).abs() <= po.bound(ref, mass, size, D, n[b], dtype)).all()
    rk, _ = c.read()
    assert rk.dtype == dtype and rk.shape == (B, H, 100, D) and (rk[1, :, n[1]:] == 0).all()
    if kv is None:
        for b in range(B):
            assert torch.equal(rk[b, :, :counts[b]], k[b, :, :counts[b]])
            assert torch.equal(rk[b, :, counts[b]:counts[b] + 5], k[b, :, :5])


def test_sequences_that_are_not_in_use(gpu_device):
    """At a negative position nothing is written, steps give zeros and the position stays; the others go on."""
    B, H, D = 3, 2, 64
    g = torch.Generator().manual_seed(7)
    c, only = PagedKVCache(B, H, D, 40, BF, gpu_device, page_size=16), PagedKVCache(B, H, D, 40, BF, gpu_device, page_size=16)
    k, v = (torch.randn(B, H, 9, D, generator=g).to(gpu_device, BF) for _ in range(2))
    for x in (c, only):
        x.prefill(k, v)
    c.pos[1] = -1
    c.write(k[:, :, :4], v[:, :, :4])
    only.write(k[:, :, :4], v[:, :, :4])
    assert c.pos.tolist() == [13, -1, 13]
    c.write(k[:, :, :4], v[:, :, :4], torch.tensor([2, 3, 0], device=gpu_device))
    only.write(k[:, :, :4], v[:, :, :4], torch.tensor([2, 0, 0], device=gpu_device))
    assert c.pos.tolist() == [15, -1, 13]
    for i in range(3):
        q, kt, vt = (torch.randn(B, H, D, generator=g).to(gpu_device, BF) for _ in range(3))
        a, b = c.step(q, kt, vt), only.step(q, kt, vt)
        same(a[0], b[0])
        same(a[2], b[2])
        assert (a[1] == 0).all() and c.pos.tolist() == [16 + i, -1, 14 + i]
    assert torch.equal(c.k_pages[3:6, :, 9:], torch.zeros_like(c.k_pages[3:6, :, 9:]))
    assert torch.equal(c.k_pages[3, :, :9], k[1])


def _model(dev, dtype):
    torch.manual_seed(0)
    m = dwarf_amd.CondMTransformer(101, 64, 3, 2, 128, 96, full_attn_layer=1, interference_interval=3)
    for p in m.parameters():
        p.data.mul_(3.0)
    return m.to(dev, dtype).eval()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_model_with_a_paged_cache(gpu_device, dtype):
    """Prefill and steps of the model: the logits of its flat cache, to the type's rounding."""
    m = _model(gpu_device, dtype)
    ids = torch.randint(0, 101, (2, 40), generator=torch.Generator().manual_seed(3)).to(gpu_device)
    flat, paged = m.new_cache(2), m.new_cache(2, paged=True)
    assert isinstance(paged.blocks[1], PagedKVCache) and paged.blocks[1].k_pages.dtype == dtype
    with torch.no_grad():
        assert torch.equal(m.prefill(ids[:, :30], flat), m.prefill(ids[:, :30], paged))
    with pytest.raises(RuntimeError):  # a step past the caller's own grad mode is not the point here
        dwarf_amd.paged_decode_step(*(torch.zeros(2, 2, 32, device=gpu_device, dtype=dtype).requires_grad_(),) * 3,
                                    paged.blocks[1].k_pages, paged.blocks[1].v_pages, paged.blocks[1].page_table,
                                    paged.blocks[1].pos)
    for t in range(30, 40):
        a, b = m.step(ids[:, t], flat), m.step(ids[:, t], paged)
        # The layers behind the attention carry its rounding (one step of the type) on, to a few steps.
        assert (a - b).abs().max() <= 16 * torch.finfo(dtype).eps * a.abs().max()
    assert paged.blocks[1].pos.tolist() == [40, 40]
    k, v = paged.blocks[1].read()
    assert (k[:, :, :30] - flat.blocks[1].k[:, :, :30]).abs().max() == 0


@pytest.mark.parametrize("use_graph", [True, False])
def test_generation_with_a_paged_cache(gpu_device, use_graph):
    """Greedy tokens of the flat cache, past the position table too; an 8-bit cache runs the same way."""
    m = _model(gpu_device, F32)
    ids = torch.randint(0, 101, (2, 20), generator=torch.Generator().manual_seed(4)).to(gpu_device)
    want = m.generate(ids, 80, temperature=0.0, use_graph=use_graph)
    assert torch.equal(m.generate(ids, 80, temperature=0.0, use_graph=use_graph, paged=True), want)
    for kv in (E4, I8):
        got = m.generate(ids, 12, temperature=0.0, use_graph=use_graph, kv_dtype=kv)
        assert got.shape == (2, 32) and torch.equal(got[:, :21], want[:, :21])


def test_prefill_records_no_gradient_in_the_cache(gpu_device):
    block = dwarf_amd.FullAttentionBlock(64, 2, 128).to(gpu_device)
    cache = block.new_cache(1, 32, paged=True)
    x = torch.randn(1, 10, 64, device=gpu_device, requires_grad=True)
    y = block.prefill(x, cache)
    assert y.requires_grad and not cache.k_pages.requires_grad
    y.sum().backward()
    assert x.grad is not None


# ---- Infinite values of little weight. ----------------------------------------------------------------------------

@pytest.mark.parametrize("drop", [5.0, 20.0, 26.0, 30.0, 60.0])
@pytest.mark.parametrize("dtype,G", [(F16, 1), (F16, 4), (F16, 16), (BF, 1), (BF, 8), (F32, 1), (F32, 4)])
def test_step_infinite_values_of_little_weight(gpu_device, dtype, G, drop):
    """An infinity in a row whose score lies far below the largest is that infinity (times a weight above zero),
    and the other columns are what they are without it."""
    n, D = 150, 64
    c = Cache(gpu_device, 1, 1, D, 16, 10, dtype)
    at = int(c.table[0, 70 // 16]), 0, 70 % 16
    c.k.zero_()
    c.k[at] = -drop / 8  # times 64 ones and a scale of 1/8: a score of -drop
    q = torch.ones(1, G, D, device=gpu_device, dtype=dtype)
    pos = torch.tensor([n - 1], device=gpu_device)
    plain = paged_decode_step(q, None, None, c.k, c.v, c.table, pos)
    c.v[at][7], c.v[at][40] = math.inf, -math.inf
    out = paged_decode_step(q, None, None, c.k, c.v, c.table, pos)
    assert (out[:, :, 7] == math.inf).all() and (out[:, :, 40] == -math.inf).all()
    rest = [d for d in range(D) if d not in (7, 40)]
    same(out[:, :, rest], plain[:, :, rest])


# ---- Large scores. --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("dtype,kv", [(F16, None), (BF, None), (F32, None), (BF, E4), (BF, I8), (F16, E4), (F16, I8), (F32, I8)])
def test_step_large_scores(gpu_device, dtype, kv, fresh, G):
    """Scores far past 2^24, where a rounding is larger than any softmax's range: the largest one's row has all
    the weight, be it a stored one or the new one."""
    n, D = 150, 64
    for c0 in (3e2, 1e3, 3e3, 1.7e4, 4e4) + ((3e5, 1e6, 7e7, 1e10, 1e15) if dtype != F16 else ()):
        for at in (3, 70, n - 1):
            c = PagedKVCache(1, 1, D, 160, dtype, gpu_device, kv_dtype=kv, page_size=16)
            k = torch.full((1, 1, n, D), -c0, device=gpu_device)
            k[:, :, at] = c0
            v = torch.randn(1, 1, n, D, generator=torch.Generator().manual_seed(at)).to(gpu_device, dtype)
            k, q = k.to(dtype), torch.full((1, G, D), c0, device=gpu_device).to(dtype)
            c.prefill(k[:, :, :n - fresh], v[:, :, :n - fresh])
            out = c.step(q, k[:, :, -1], v[:, :, -1]) if fresh else \
                paged_decode_step(q, None, None, c.k_pages, c.v_pages, c.page_table, c.pos - 1, k_scale=c.k_scale, v_scale=c.v_scale)
            want = c.read(dtype=F32)[1][0, 0, at].expand(G, D)
            # One row's value, its weight in two 16-bit terms at worst (2^-16), then rounded to the type.
            err = (out[0].float() - want).abs()
            assert (err <= want.abs() * (2.0 ** -16 + torch.finfo(dtype).eps / 2)).all(), (c0, at)


# ---- Operands that count as contiguous. --------------------------------------------

def _odd_base(t, by=4):
    """t at an address that is no multiple of 16 bytes, contiguous as it was."""
    flat = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    out = flat[by if t.element_size() == 2 else by // 2:][:t.numel()].view(t.shape)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out.copy_(t)


def _odd_ones(t):
    """t with a stride of 3 elements in its dimensions of one entry (which count for nothing)."""
    strides = [3 if n == 1 else s for n, s in zip(t.shape, t.stride())]
    out = torch.empty(t.numel() + 64, dtype=t.dtype, device=t.device).as_strided(t.shape, strides)
    return out.copy_(t)


@pytest.mark.parametrize("form", [_odd_base, _odd_ones])
@pytest.mark.parametrize("B,H,N", [(1, 12, 5), (2, 12, 5), (1, 3, 1), (2, 1, 5), (2, 3, 1), (1, 1, 1)])
@pytest.mark.parametrize("dtype,kv", [(BF, None), (F32, None), (F16, I8)])
def test_operands_that_count_as_contiguous(gpu_device, dtype, kv, B, H, N, form):
    """Rows whose base or whose idle strides are odd: the results of aligned copies."""
    g = torch.Generator().manual_seed(8)
    rows = [torch.randn(B, H, N, 64, generator=g).to(gpu_device, dtype) for _ in range(2)]
    step = [torch.randn(B, h, 64, generator=g).to(gpu_device, dtype) for h in (2 * H, H, H)]
    pos = torch.tensor([9, 30][:B], device=gpu_device)
    res = []
    for put in (lambda t: t, form):
        c = Cache(gpu_device, B, H, 64, 16, 3, dtype, kv)
        paged_kv_write(*(put(t) for t in rows), c.k, c.v, c.table, pos, **c.state)
        out = paged_decode_step(*(put(t) for t in step), c.k, c.v, c.table, pos + N, **c.state)
        res.append([out, c.k, c.v, *(s for s in (c.k_scale, c.v_scale) if s is not None)])
    for a, b in zip(*res):
        same(a, b)


def _odd_pool(t):
    u = t.view(torch.uint8) if t.element_size() == 1 else t
    strides = [3 if n == 1 else s for n, s in zip(u.shape, u.stride())]
    return u.clone().as_strided(u.shape, strides).view(t.dtype)


@pytest.mark.parametrize("P,H", [(1, 2), (5, 1), (1, 1)])
@pytest.mark.parametrize("kv", [None, E4])
def test_pools_with_idle_strides(gpu_device, kv, P, H):
    """A pool of one page or one head may have any stride there."""
    g = torch.Generator().manual_seed(8)
    row = [torch.randn(1, h, 32, generator=g).to(gpu_device, BF) for h in (3 * H, H, H)]
    pos = torch.tensor([7], device=gpu_device)
    res = []
    for put in (lambda t: t, _odd_pool):
        c = Cache(gpu_device, 1, H, 32, 16, 1, BF, kv, spare=P - 1)
        c.k, c.v = put(c.k), put(c.v)
        if kv is not None:
            c.k_scale, c.v_scale = put(c.k_scale), put(c.v_scale)
        out = paged_decode_step(*row, c.k, c.v, c.table, pos, **c.state)
        paged_kv_write(row[1][:, :, None], row[2][:, :, None], c.k, c.v, c.table, pos + 1, **c.state)
        res.append([out, *paged_kv_read(c.k, c.v, c.table, pos + 2, 16, **c.state)])
    for a, b in zip(*res):
        same(a, b)


# ---- Calls of more rows than one grid has. ------------------------------------------------------------------------

def test_read_of_more_rows_than_a_grid(gpu_device):
    """2^27 rows of a sequence and a few: pages come round again and again, so that every row is known."""
    H, D, page = 8, 32, 65536
    T = 2 ** 24 + 70000
    M = -(-T // page)
    g = torch.Generator(gpu_device).manual_seed(1)
    k, v = (torch.randn(3, H, page, D, device=gpu_device, dtype=BF, generator=g) for _ in range(2))
    table = (torch.arange(M, device=gpu_device) % 3).to(torch.int32)[None]
    n = T - 300
    got = paged_kv_read(k, v, table, torch.tensor([n], device=gpu_device), T)
    for x, pool in zip(got, (k, v)):
        assert x.shape == (1, H, T, D)
        for j in range(M):
            live = min(page, n - j * page)
            if live > 0:
                assert torch.equal(x[0, :, j * page:j * page + live], pool[j % 3, :, :live]), j
        assert not x[0, :, n:].any()


def test_write_of_more_rows_than_a_grid(gpu_device):
    """The last rows of the last head lie behind the 2^27th; those in front of the sequence are left out."""
    H, D, N = 8, 32, 2 ** 24 + 5
    g = torch.Generator(gpu_device).manual_seed(1)
    k = torch.randn(1, H, N, D, device=gpu_device, dtype=BF, generator=g)
    v = k.flip(-1)
    kp, vp = (torch.zeros(2, H, 64, D, device=gpu_device, dtype=BF) for _ in range(2))
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=gpu_device)
    paged_kv_write(k, v, kp, vp, table, torch.tensor([100 - N], device=gpu_device))
    for pool, x in ((kp, k), (vp, v)):
        same(pool[1], x[0, :, N - 100:N - 36])
        same(pool[0, :, :36], x[0, :, N - 36:])
        assert not pool[0, :, 36:].any()


# ---- Equal shares of wide rows. -----------------------------------------------------------------------------------

@pytest.mark.parametrize("B,H,G,most", [(12, 4, 3, 12000), (64, 16, 1, 260), (3, 8, 16, 30000)])
@pytest.mark.parametrize("dtype,kv", [(BF, E4), (BF, I8), (F16, E4), (F16, I8)])
def test_step_shares_of_wide_rows(gpu_device, dtype, kv, B, H, G, most):
    """128 elements in 8 bits: units of several shares, shares of several units, sequences without rows."""
    from test_paged_cpu import split_of
    g = torch.Generator().manual_seed(B)
    pos = (torch.rand(B, generator=g) ** 2 * most).long().tolist()
    pos[0], pos[1], pos[2] = most, -1, 128
    if B > 3:
        pos[-1], pos[-2] = 255, 256
    M = 16 * 768 * 128 // (B * H * 32) * 2 + 1024
    c = RaggedCache(gpu_device, H, 128, 32, M, dtype, kv, [p + 1 for p in pos])
    assert split_of(dtype, kv, B, H, H * G, 128, 32, M)[0] == "shares"
    junk(c, [p + 1 for p in pos])
    if B > 3:
        pos[3] = M * 32 + 5  # past the table
    for fresh in (True, False):
        a = _step(c, pos, G, fresh)
    same(_step(c, pos, G, False), a)


# ---- The range of values that the step keeps. -------------------------------------------------------------------------

@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("dtype,kv,e", [(BF, None, -90), (F32, None, -90), (BF, E4, -70), (BF, I8, -70), (F32, E4, -70), (F32, I8, -70),
                                        (BF, None, 126), (F32, None, 126), (BF, E4, 126), (F32, I8, 126)])
def test_step_small_and_large_values(gpu_device, dtype, kv, e, G):
    """Values near the ends of the stated range, under weights of all sizes, within the bound that holds elsewhere."""
    n, D = 700, 64
    g = torch.Generator().manual_seed(2)
    c = PagedKVCache(2, 2, D, n, dtype, gpu_device, kv_dtype=kv, page_size=16)
    k, v = (torch.randn(2, 2, n, D, generator=g) for _ in range(2))
    # Rows whose largest magnitude is from 2^e to 2^(e + 1).
    v = v / v.abs().amax(-1, keepdim=True) * 2.0 ** e * (1 + torch.rand(2, 2, n, 1, generator=g))
    k, v = k.to(gpu_device, dtype), v.to(gpu_device, dtype)
    c.prefill(k, v)
    q = (torch.randn(2, 2 * G, D, generator=g) * 2).to(gpu_device, dtype)
    out = paged_decode_step(q, None, None, c.k_pages, c.v_pages, c.page_table, c.pos - 1, k_scale=c.k_scale, v_scale=c.v_scale)
    rk, rv = c.read(dtype=F32)
    for b in range(2):
        ref, mass, size = po.attend(q[b].cpu(), rk[b].cpu().double(), rv[b].cpu().double(), D ** -0.5)
        assert ((out[b].double().cpu() - ref).abs() <= po.bound(ref, mass, size, D, n, dtype)).all()


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
@pytest.mark.parametrize("dtype,kv,G", [(BF, None, 1), (F16, None, 4), (BF, E4, 4), (F16, I8, 3), (F32, I8, 2)])
def test_step_softmax_scale_of_narrow_types(gpu_device, dtype, kv, G, scale):
    """A flat softmax, a sharp one and a reversed one, with and without a new row, in one part and in several."""
    for pos, M in (([300, 45], 5), ([3000, 129], 60)):
        for fresh in (True, False):
            c = Cache(gpu_device, 2, 2, 64, 64, M, dtype, kv, [p + 1 for p in pos])
            junk(c, [p + 1 for p in pos])
            _step(c, pos, G, fresh, scale=scale)
