"""Sampling and the walk over drafted tokens on the GPU against the 64-bit oracle: tokens are equal wherever u and the
nucleus' limit lie further from a border than the masses' rounding."""

import math

import pytest
import torch

from dwarf_amd import draft_tree_accept, paged_kv_read, paged_kv_write, sample_tokens
from oracle import sample_oracle as so

pytestmark = pytest.mark.gpu
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, dev="cuda:0"):
    """Every row of x (CPU, any layout) against the oracle.  A mass is rounded by at most half of 2^-F of the largest, so
    a running sum over V of them is off by V 2^-(F+1) <= 2^-33 of the total (F = 62 - log2 V beyond 2^14 tokens, so
    V 2^-F = 2^(2 log2 V - 62) < 2^-24 for the 2^18 tokens and less used here), the exponentials by about 2^-50."""
    B, V = x.shape
    tol = max(2.0 ** -33, V * 2.0 ** -(48 if V <= 1 << 14 else 62 - (V - 1).bit_length()))

    def gpu(s):
        return s.to(dev) if torch.is_tensor(s) else s

    def row(s, b):
        return s[b].item() if torch.is_tensor(s) else s

    tokens, logp = sample_tokens(x.to(dev), u.to(dev), gpu(temperature), gpu(top_k), gpu(top_p), gpu(min_p), return_logprobs=True)
    again = sample_tokens(x.to(dev), u.to(dev), gpu(temperature), gpu(top_k), gpu(top_p), gpu(min_p))
    assert torch.equal(tokens, again)
    tokens, logp, near = tokens.cpu(), logp.cpu().double(), 0
    xs = x.double()
    for b in range(B):
        t, lp, margin = so.sample(xs[b].tolist(), row(u, b), row(temperature, b), row(top_k, b), row(top_p, b), row(min_p, b))
        if margin <= tol:
            near += 1
            continue
        assert tokens[b].item() == t, f"row {b}: token {tokens[b].item()}, oracle {t}"
        # log w - log K in 64 bits, rounded to float32: half a step, and the masses' rounding.
        assert logp[b] == lp or abs(logp[b] - lp) <= 2.0 ** -24 * abs(lp) + 2 * tol, (logp[b].item(), lp)
    # (Without a temperature all weights are equal, and 0.3 of 300 of them ends at a border in every row.)
    assert near <= B // 4 + 1 or temperature == math.inf


def rows(B, V, seed, dtype=F32, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, V, generator=g) * scale).to(dtype), torch.rand(B, generator=g)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 257, 1000, 4099, 32000])
def test_sizes(gpu_device, dtype, V):
    B = 9 if V < 10000 else 3
    x, u = rows(B, V, V, dtype)
    check(x, u)
    check(x, u, 0.7, top_k=5, top_p=0.9, min_p=0.02)
    check(x, u, 1.3, top_p=0.5)
    check(x, u, 0.9, top_k=40)


@pytest.mark.parametrize("temperature", [0.0, 1e-30, 1e-3, 0.3, 1.0, 30.0, 1e6, math.inf])
@pytest.mark.parametrize("kw", [dict(), dict(top_p=0.6), dict(top_k=11), dict(top_k=300, top_p=0.3), dict(min_p=0.3),
                                dict(top_p=0.0), dict(top_k=1), dict(min_p=1.0)])
def test_temperatures(gpu_device, temperature, kw):
    for dtype in (F32, BF):
        x, u = rows(6, 777, 3, dtype)
        check(x, u, temperature, **kw)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_settings_of_each_row(gpu_device, dtype):
    B, V = 40, 1500
    x, u = rows(B, V, 11, dtype)
    g = torch.Generator().manual_seed(5)
    t = torch.rand(B, generator=g) * 1.5
    t[::6] = torch.tensor([0.0, -1.0, math.nan, 0.0, 1.0, 2.0, 0.1])
    k = torch.randint(-3, 60, (B,), generator=g)
    k[7], k[8] = V, 2 ** 40
    p = torch.rand(B, generator=g) * 1.2 - 0.1
    p[3] = math.nan
    m = torch.rand(B, generator=g) * 0.3 - 0.1
    m[4], m[5] = math.nan, 7.0
    # As the oracle reads them: a NaN temperature is greedy, a NaN limit none.
    tokens, logp = sample_tokens(x.to("cuda:0"), u.to("cuda:0"), t.to("cuda:0"), k.to("cuda:0"), p.to("cuda:0"), m.to("cuda:0"),
                                 return_logprobs=True)
    for b in range(B):
        want, lp, margin = so.sample(x[b].double().tolist(), u[b].item(), t[b].item(), k[b].item(), 1.0 if b == 3 else p[b].item(),
                                     0.0 if b == 4 else m[b].item())
        if margin > 2.0 ** -33:
            assert tokens[b].item() == want and (abs(logp[b].item() - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -32)
    # Other types of the same numbers.
    a = sample_tokens(x.to("cuda:0"), u.to("cuda:0"), 0.75, k.int().clamp(0).to("cuda:0"), p.double().to("cuda:0"))
    b = sample_tokens(x.to("cuda:0"), u.to("cuda:0"), torch.full((B,), 0.75, device="cuda:0"), k.clamp(0).to("cuda:0"), p.to("cuda:0"))
    assert torch.equal(a, b)


def test_ties(gpu_device):
    """Equal logits: limits that end inside a group keep its first by index."""
    V = 5000
    for x in (torch.zeros(1, V), (torch.arange(V) % 7).float()[None], (torch.arange(V) % 3).float()[None] * 1e-7,
              torch.full((1, V), 3.0e38), torch.full((1, V), torch.finfo(F32).min), torch.zeros(1, V).index_fill(1, torch.arange(100, 200), -0.0)):
        for kw in (dict(), dict(top_k=1), dict(top_k=3), dict(top_k=2345), dict(top_p=0.37), dict(top_k=1000, top_p=0.731), dict(min_p=0.9)):
            for u in (0.0, 0.1234567, 0.5001, 0.99999):
                check(x, torch.tensor([u]), **kw)
    check(torch.zeros(1, V, dtype=BF), torch.tensor([0.31]), top_p=0.4217)


def test_close_values(gpu_device):
    """Logits a few units in the last place apart, more of them than the list in LDS holds."""
    base = torch.tensor([5.0]).view(torch.int32)
    for n in (700, 9000):
        g = torch.Generator().manual_seed(n)
        x = (base + torch.randint(0, 40, (3, n), generator=g, dtype=torch.int32)).view(F32)
        for kw in (dict(top_k=n // 3), dict(top_p=0.4123), dict(top_k=n // 2, top_p=0.7), dict(top_k=n - 1)):
            for t in (1.0, 1e-6):
                check(x, torch.rand(3, generator=g), t, **kw)


def test_special_values(gpu_device):
    inf, nan = math.inf, math.nan
    low = torch.finfo(F32).min
    x = torch.tensor([[nan, 1.0, -inf, 2.0, nan, 0.5, -inf, 1.0], [-inf] * 8, [nan] * 8, [inf, 1.0, nan, inf, -inf, 0.0, inf, 3.0],
                      [-inf, -inf, 0.0, -inf, -inf, -inf, -inf, -inf], [low] * 8, [low, 1.0, low, 2.0, low, low, low, low],
                      [1e38, -1e38, 3e38, -3e38, 0.0, 1.0, 2.0, 3e38]])
    for u in (0.0, 0.3, 0.7, 0.999):
        for kw in (dict(), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.5), dict(temperature=0.0), dict(temperature=2.0, top_k=3, top_p=0.9)):
            check(x, torch.full((8,), u), **kw)
    for dtype in (BF, F16):
        y = x.to(dtype)
        check(y, torch.full((8,), 0.7), top_p=0.9)


def test_uniform_numbers_at_the_ends(gpu_device):
    x, _ = rows(6, 300, 2)
    u = torch.tensor([0.0, -0.0, -1.0, 1.0, 2.0, math.nan])
    t = sample_tokens(x.to("cuda:0"), u.to("cuda:0"), top_p=0.5).cpu()
    for b in range(6):
        lo, hi = so.sample(x[b].double().tolist(), 0.0, top_p=0.5)[0], so.sample(x[b].double().tolist(), 1.0, top_p=0.5)[0]
        assert t[b].item() == (hi if b in (3, 4) else lo)
    # 64-bit numbers are taken as they are.
    y = torch.zeros(1, 1 << 16)
    for k in (1, 12345, 65535):
        u = torch.tensor([k / 65536 - 2.0 ** -40], dtype=torch.float64)
        assert sample_tokens(y.to("cuda:0"), u.to("cuda:0")).item() == k - 1
        u = torch.tensor([k / 65536], dtype=torch.float64)
        assert sample_tokens(y.to("cuda:0"), u.to("cuda:0")).item() == k


def test_layouts(gpu_device):
    B, V = 5, 333
    base, u = rows(B, 3 * V + 5, 4)
    for dtype in (F32, BF):
        wide = base.to(dtype).to("cuda:0")
        want = sample_tokens(wide[:, 7:7 + V].contiguous(), u.to("cuda:0"), top_p=0.8)
        ux = u.to("cuda:0")
        assert torch.equal(sample_tokens(wide[:, 7:7 + V], ux, top_p=0.8), want)                       # misaligned rows
        assert torch.equal(sample_tokens(wide[:, 7:7 + V].t().contiguous().t(), ux, top_p=0.8), want)  # columns
        assert torch.equal(sample_tokens(torch._neg_view(-wide[:, 7:7 + V]), ux, top_p=0.8), want)
        x3 = wide[:4, 7:7 + V].reshape(2, 2, V)
        assert torch.equal(sample_tokens(x3, ux[:4].view(2, 2), top_p=0.8), want[:4].view(2, 2))
        assert torch.equal(sample_tokens(wide[:1, 7:7 + V].expand(3, V), ux[:1].expand(3), top_p=0.8), want[:1].expand(3))
        assert sample_tokens(wide[0, 7:7 + V], ux[0], top_p=0.8) == want[0]
        assert sample_tokens(wide[:0, :V], ux[:0]).shape == (0,)


def test_neighbours_are_not_read(gpu_device):
    """Rows start and end inside 16-byte pieces whose other elements are larger than any of the row's."""
    for dtype in (F32, BF, F16):
        big = torch.full((4, 64), math.inf, dtype=dtype, device="cuda:0")
        for at in range(9):
            for n in (1, 3, 8, 17):
                big.fill_(math.inf)
                big[:, at:at + n] = torch.arange(n, device="cuda:0").to(dtype)
                t, lp = sample_tokens(big[:, at:at + n], torch.full((4,), 0.999999, device="cuda:0"), return_logprobs=True)
                assert (t == n - 1).all() and (lp <= 0).all()


def test_graph_and_streams(gpu_device):
    x, u = rows(8, 5003, 21)
    x, u = x.to("cuda:0"), u.to("cuda:0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sample_tokens(x, u, 0.8, 40, 0.9, return_logprobs=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t, lp = sample_tokens(x, u, 0.8, 40, 0.9, return_logprobs=True)
    for seed in range(4):
        y, v = rows(8, 5003, seed)
        x.copy_(y)
        u.copy_(v)
        graph.replay()
        want = sample_tokens(x, u, 0.8, 40, 0.9, return_logprobs=True)
        torch.cuda.synchronize()
        assert torch.equal(t, want[0]) and torch.equal(lp, want[1])


def test_traced_call(gpu_device):
    x, u = rows(4, 500, 8)
    x, u = x.to("cuda:0"), u.to("cuda:0")
    f = torch.compile(lambda a, b: sample_tokens(a * 2.0, b, 0.9, top_k=7, return_logprobs=True), backend="eager")
    a, b = f(x, u), sample_tokens(x * 2.0, u, 0.9, top_k=7, return_logprobs=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- Drafted trees. ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T", [1, 2, 5, 31, 63, 64])
@pytest.mark.parametrize("shared", [True, False])
def test_walk(gpu_device, T, shared):
    B = 50
    g = torch.Generator().manual_seed(T)
    parents = torch.stack([torch.randint(0, max(1, i), (B,), generator=g) for i in range(T)], 1)
    parents[:, 0] = -1
    if shared:
        parents = parents[:1].expand(B, T)
    tokens = torch.randint(0, 3, (B, T), generator=g)  # few tokens: siblings often have the same
    picks = torch.randint(0, 3, (B, T), generator=g)
    tokens[0], picks[0] = 2 ** 40, 2 ** 40             # the whole chain of first children, past 32 bits
    counts = torch.randint(-1, T + 3, (B,), generator=g)
    for c in (None, counts):
        for pt in (torch.int32, torch.int64):
            p = (parents[0] if shared else parents).to(pt).to("cuda:0")
            path, n, nxt = draft_tree_accept(tokens.to("cuda:0"), p, picks.to("cuda:0"), None if c is None else c.to("cuda:0"))
            for b in range(B):
                want, last = so.walk(tokens[b].tolist(), parents[b].tolist(), picks[b].tolist(), None if c is None else c[b].item())
                assert path[b].tolist() == want + [-1] * (T - len(want)) and n[b].item() == len(want) and nxt[b].item() == last


def test_walk_over_no_tree(gpu_device):
    """Parents that are no earlier node end at themselves: no step goes back or stays."""
    z = torch.zeros(2, 6, dtype=torch.int64, device="cuda:0")
    parents = torch.tensor([[5, 1, 0, 3, 2, 0], [0, 0, 99, -7, 1, 4]], device="cuda:0")
    path, n, nxt = draft_tree_accept(z, parents, z)
    assert path.tolist() == [[0, 2, 4, -1, -1, -1], [0, 1, 4, 5, -1, -1]] and n.tolist() == [3, 4] and nxt.tolist() == [0, 0]
    assert draft_tree_accept(z[:0], parents[0], z[:0])[0].shape == (0, 6)
    s = torch.arange(24, device="cuda:0").view(2, 12)[:, ::2]  # strided tokens
    path, n, _ = draft_tree_accept(s, parents, s.roll(-1, 1))
    assert n.tolist() == draft_tree_accept(s.contiguous(), parents, s.roll(-1, 1).contiguous())[1].tolist()


@pytest.mark.parametrize("kv", [BF, torch.float8_e4m3fn, torch.int8])
def test_write_rows(gpu_device, kv):
    """Rows by number are what the same rows, gathered first, are; numbers of no row leave the pages alone."""
    dev, B, H, N, D, page = "cuda:0", 3, 2, 7, 64, 16
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(B, N, H, D, generator=g).to(BF).to(dev).permute(0, 2, 1, 3) for _ in range(2))
    rows = torch.tensor([[0, 2, 5, -1, -1], [6, 6, 0, 1, 3], [7, 0, 2 ** 40, -5, 4]], device=dev)
    table = torch.randperm(9, generator=g).to(torch.int32).view(3, 3).to(dev)
    pos = torch.tensor([14, 0, 30], device=dev)
    counts = torch.tensor([3, 5, 5], device=dev)

    def pools():
        if kv == BF:
            return torch.zeros(9, H, page, D, dtype=BF, device=dev), torch.zeros(9, H, page, D, dtype=BF, device=dev), {}
        z = [torch.zeros(9, H, page, D, dtype=kv, device=dev) for _ in range(2)]
        return *z, {n: torch.zeros(9, H, page, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu) for n in ("k_scale", "v_scale")}

    a, b = pools(), pools()
    paged_kv_write(k, v, a[0], a[1], table, pos, counts=counts, rows=rows, **a[2])
    for s in range(B):
        for i, r in enumerate(rows[s].tolist()):
            if i < counts[s] and 0 <= r < N:
                at = torch.full((B,), 10 ** 6, device=dev)  # (others go past the table)
                at[s] = pos[s] + i
                paged_kv_write(k[:, :, r:r + 1], v[:, :, r:r + 1], b[0], b[1], table, at, **b[2])
    for x, y in zip(a[:2], b[:2]):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    for n in a[2]:
        assert torch.equal(a[2][n].view(torch.uint8), b[2][n].view(torch.uint8))
    # No rows at all.
    c = pools()
    paged_kv_write(k[:, :, :0], v[:, :, :0], c[0], c[1], table, pos, rows=rows, **c[2])
    paged_kv_write(k, v, c[0], c[1], table, pos, rows=rows[:, :0], **c[2])
    assert not c[0].view(torch.uint8).any()


@pytest.mark.parametrize("V,dtype", [(8192, F32), (9001, BF), (40001, F16), (40000, F32)])
def test_split_rows(gpu_device, V, dtype):
    """A few long rows, which several workgroups share: every way that the limits take, row by row and together."""
    x, u = rows(5, V + 3, V, dtype)
    x[1, :] = 0.25                          # equal logits, whose limits end inside a group
    x[2, torch.arange(V + 3) % 997 != 5] = -math.inf  # a masked vocabulary
    x[3, 100:V:50] = math.nan
    x = x[:, 3:]                            # (rows that begin anywhere)
    for kw in (dict(), dict(top_k=1), dict(top_k=50, top_p=0.8), dict(top_k=1000, min_p=0.01), dict(top_k=1500, top_p=0.9),
               dict(top_p=0.9), dict(top_p=0.99999), dict(min_p=0.05), dict(temperature=0.0)):
        check(x, u, **{"temperature": 0.8, **kw})
    k, p = torch.tensor([0, 7, 3, 2000, V]), torch.tensor([0.7, 1.0, 0.5, 0.9, 1.0])
    t = torch.tensor([0.9, 1.1, 0.0, 0.7, math.inf])
    check(x, u, t, k, p, torch.tensor([0.0, 0.0, 0.1, 0.002, 0.0]))
    y = x.clone()
    y[0, V // 2] = y[0, V - 1] = math.inf   # infinities share their row
    y[4] = -math.inf                        # no candidate
    check(y, u, 0.9, top_p=0.95)
    check(y, u, 0.9, top_k=11)


def test_split_rows_in_two_graphs(gpu_device):
    """Graphs that are replayed in turn, each with scratch memory of its own."""
    x, u = rows(2, 50000, 3)
    x, u = x.cuda(), u.cuda()
    y, v = x.flip(1).contiguous(), 1 - u
    calls = [lambda: sample_tokens(x, u, 0.9, top_p=0.9, return_logprobs=True), lambda: sample_tokens(y, v, 1.1, top_k=30, return_logprobs=True)]
    graphs, outs = [], []
    for call in calls:
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for i in range(4):
        x.copy_(torch.randn(2, 50000, generator=torch.Generator().manual_seed(50 + i)) * 2)
        y.copy_(x.flip(1))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for call, out in zip(calls, outs):
            for a, b in zip(call(), out):
                assert torch.equal(a, b)


def test_many_of_few(gpu_device):
    """A top-k of most of a row that the list holds, and rows a little longer than it."""
    for V, k in ((3000, 2000), (4096, 1025), (4097, 1024), (6000, 1024)):
        for dtype in (F32, BF):
            x, u = rows(6, V, V + k, dtype)
            check(x, u, 0.9, top_k=k)
            check(x, u, 0.6, top_k=k, top_p=0.97, min_p=1e-4)
