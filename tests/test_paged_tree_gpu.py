"""Steps of drafted tokens over the paged cache against the 64-bit oracle: trees of every size and shape, windows with
sinks, types, layouts, what stands in places that a node does not see, refusals, captured and traced calls."""

import math
import random

import pytest
import torch

import dwarf_amd
from dwarf_amd import PagedKVCache, draft_tree_accept, paged_decode_step, paged_kv_read, paged_tree_step
from oracle import paged_oracle as po
from tests.test_paged_gpu import Cache, _expect_write, junk, same

pytestmark = pytest.mark.gpu
F32, BF, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


def tree(T, seed, kind="random"):
    rng = random.Random(seed)
    if kind == "chain":
        return list(range(-1, T - 1))
    if kind == "star":
        return [-1] + [0] * (T - 1)
    if kind == "forest":  # several roots
        return [rng.choice([-1, rng.randrange(-1, i)]) if i else -1 for i in range(T)]
    if kind == "broken":  # nodes that hang on none, on later ones or on themselves
        p = [rng.randrange(-1, max(1, i)) for i in range(T)]
        for i in rng.sample(range(T), max(1, T // 5)):
            p[i] = rng.choice([i, i + 1, T + 5, -2, -2 ** 31, 2 ** 31 - 1])
        return p
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, T)]


def step(c, pos, parents, G=1, counts=None, window=None, sinks=0, fresh=True, scale=None, seed=3, shared=False,
         layout="tokens", kv=None):
    """Runs a step and checks its output and the rows that it wrote.  parents: a list for each sequence, or None."""
    B, (P, H, page, D), dev = len(pos), c.k.shape, c.dev
    T = len(parents[0]) if parents is not None else kv
    g = torch.Generator().manual_seed(seed)

    def rows(heads):
        if layout == "tokens":  # head views of a projection's output
            return torch.randn(B, T, heads, D, generator=g).to(dev, c.dtype).permute(0, 2, 1, 3)
        if layout == "unaligned":
            return torch.randn(B, heads, T, D + 1, generator=g).to(dev, c.dtype)[..., 1:]
        return torch.randn(B, heads, T, D, generator=g).to(dev, c.dtype)

    q = rows(H * G) * 2 if layout != "tokens" else (torch.randn(B, T, H * G, D, generator=g) * 2).to(dev, c.dtype).permute(0, 2, 1, 3)
    kn, vn = (rows(H), rows(H)) if fresh else (None, None)
    have = [T if counts is None else max(0, min(T, counts[b])) if pos[b] >= 0 else 0 for b in range(B)]
    have = [n if pos[b] >= 0 else 0 for b, n in enumerate(have)]
    if fresh:
        want = _expect_write(c, kn, vn, pos, have)
    else:
        want = [None if t is None else c.cpu(t.contiguous()).clone() for t in (c.k, c.k_scale, c.v, c.v_scale)]
    pt = None
    if parents is not None:
        pt = torch.tensor(parents[0] if shared else parents, dtype=torch.int64).clamp(-2 ** 31, 2 ** 31 - 1).to(dev, torch.int32)
    out = paged_tree_step(q, kn, vn, c.k, c.v, c.table, torch.tensor(pos, device=dev), pt,
                          counts=None if counts is None else torch.tensor(counts, device=dev), window=window, sinks=sinks,
                          softmax_scale=scale, **c.state)
    for got, ref in zip((c.k, c.k_scale, c.v, c.v_scale), want):
        if ref is not None:
            same(got, ref)
    assert out.dtype == c.dtype and out.shape == q.shape and out.stride() == (T * H * G * D, D, H * G * D, 1)
    x = out.double().cpu()
    for b, n in enumerate(pos):
        line = list(range(-1, T - 1)) if parents is None else parents[0] if shared else parents[b]
        nodes = po.tree_rows(line, have[b])
        if n <= c.table.shape[1] * page:
            total = max(n, 0) + T
            k, v = c.rows("k", b, total), c.rows("v", b, total)
        for i, node in enumerate(nodes):
            if node is None:
                assert (x[b, :, i] == 0).all(), (b, i)
                continue
            if n > c.table.shape[1] * page:
                assert torch.isnan(x[b, :, i]).all()
                continue
            sees = po.tree_sees(node, nodes, n, window, sinks)
            kk, vv = k[:, sees], v[:, sees]
            if torch.isnan(kk).any() or torch.isnan(vv).all(-1).any():  # a position without a page
                assert torch.isnan(x[b, :, i]).all(), (b, i)
                continue
            ref, mass, size = po.attend(q[b, :, i].cpu(), kk, vv, D ** -0.5 if scale is None else scale)
            tol = po.tree_bound(ref, mass, size, D, len(sees), c.dtype, c.kv, T * G)
            err = (x[b, :, i] - ref).abs()
            assert (err <= tol).all(), f"sequence {b} node {i}: {(err / tol).max().item():.2f} of the bound"
    return out


@pytest.mark.parametrize("dtype,kv", [(F32, F32), (F32, E4), (F32, I8), (BF, BF), (BF, E4), (BF, I8), (F16, F16), (F16, E4), (F16, I8)])
@pytest.mark.parametrize("D", [32, 64, 80, 96, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (7, 2), (26, 1), (13, 5)])
def test_types_and_head_dims(gpu_device, dtype, kv, D, T, G):
    pos = [70, 0, 33]
    c = Cache(gpu_device, 3, 2, D, 16, 9, dtype, kv, [p + T for p in pos])
    junk(c, pos)
    step(c, pos, [tree(T, b) for b in range(3)], G)


@pytest.mark.parametrize("dtype,kv", [(F32, F32), (BF, BF), (F16, E4)])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 33, 63, 64])
@pytest.mark.parametrize("kind", ["random", "chain", "star", "forest", "broken"])
def test_trees(gpu_device, dtype, kv, T, kind):
    pos = [5, 100, 0, 31]
    c = Cache(gpu_device, 4, 1, 64, 32, 6, dtype, kv, [p + T for p in pos])
    junk(c, pos)
    step(c, pos, [tree(T, 10 + b, kind) for b in range(4)], shared=False)
    c = Cache(gpu_device, 4, 1, 64, 32, 6, dtype, kv, [p + T for p in pos], seed=1)
    step(c, pos, [tree(T, 3, kind)] * 4, G=2, shared=True)


@pytest.mark.parametrize("dtype,kv", [(F32, F32), (BF, BF), (BF, I8), (F16, F16)])
@pytest.mark.parametrize("window", [1, 2, 7, 40, 1000])
@pytest.mark.parametrize("sinks", [0, 1, 4, 70])
def test_windows(gpu_device, dtype, kv, window, sinks):
    pos = [0, 3, 150, 64, 95]
    for T, kind in ((1, "chain"), (12, "random"), (40, "chain")):
        c = Cache(gpu_device, 5, 2, 32, 16, 13, dtype, kv, [p + T for p in pos])
        junk(c, pos)
        step(c, pos, [tree(T, b, kind) for b in range(5)], 2, window=window, sinks=sinks)


def test_window_past_the_ends_of_integers(gpu_device):
    c = Cache(gpu_device, 2, 1, 64, 16, 4, BF)
    a = step(c, [20, 40], [tree(5, 1)] * 2)
    for w, s in ((2 ** 40, 0), (2 ** 30, 2 ** 40), (1, 2 ** 31)):
        b = step(c, [20, 40], [tree(5, 1)] * 2, window=w, sinks=s)
        assert torch.equal(a, b)


def test_given_away_pages(gpu_device):
    """Pages that a windowed step does not see may be nobody's, or hold infinities and NaN."""
    for dtype, kv in ((F32, F32), (BF, BF), (F16, F16), (BF, E4)):
        for T in (1, 9):
            c = Cache(gpu_device, 2, 2, 64, 16, 20, dtype, kv, [250 + T, 300 + T], seed=T)
            used = torch.zeros(c.P, 16, dtype=torch.bool)
            for b, n in enumerate([250, 300]):
                for t in list(range(5)) + list(range(n - 60 + 1, n)):
                    used[int(c.table[b, t // 16]), t % 16] = True
            mask = (~used).to(c.dev)[:, None, :, None]
            for x in (c.k, c.v):
                if c.narrow:
                    x.view(torch.uint8).masked_fill_(mask, 0x7f)
                else:
                    x.masked_fill_(mask, math.nan)
            for s in (c.k_scale, c.v_scale):
                if s is not None:
                    s.view(torch.uint8).masked_fill_(mask[..., 0], 255)
            c.table[:, 1:11] = -1
            step(c, [250, 300], [tree(T, 1)] * 2, 2, window=60, sinks=5)


@pytest.mark.parametrize("dtype,kv", [(F32, F32), (BF, BF), (F16, F16), (BF, E4), (F16, I8)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("T,G", [(12, 1), (30, 2)])
def test_infinities_stay_with_who_sees_them(gpu_device, dtype, kv, value, T, G):
    """A drafted row with an infinity or NaN reaches its own node and the nodes below, and no other; one in the cache,
    with a window, the nodes that see it."""
    parents = tree(T, 4)
    bad = 3
    g = torch.Generator().manual_seed(1)
    D, n = 64, 50
    for which in ("k", "v", "q", "old"):
        c = Cache(gpu_device, 1, 1, D, 16, 6, dtype, kv, [n + T])
        q, k, v = (torch.randn(1, h, T, D, generator=g).to(gpu_device, dtype) for h in (G, 1, 1))
        args = dict(q=q.clone(), k=k.clone(), v=v.clone())
        kw = dict(window=8, sinks=2) if which == "old" else {}
        pt = torch.tensor(parents, device=gpu_device)
        pos = torch.tensor([n], device=gpu_device)
        clean = paged_tree_step(args["q"], args["k"], args["v"], c.k, c.v, c.table, pos, pt, **kw, **c.state).clone()
        nodes = po.tree_rows(parents, T)
        if which == "old":
            at = n - 5
            page, slot = int(c.table[0, at // 16]), at % 16
            if c.narrow:
                c.v_scale.view(torch.uint8)[page, 0, slot] = 255
            else:
                c.v[page, 0, slot] = value
            hit = [at in po.tree_sees(nd, nodes, n, 8, 2) for nd in nodes]
            assert any(hit) and not all(hit)
        else:
            args[which][0, :, bad, 7] = value
            hit = [i == bad if which == "q" else bad in nodes[i][0] for i in range(T)]
        out = paged_tree_step(args["q"], args["k"], args["v"], c.k, c.v, c.table, pos, pt, **kw, **c.state)
        for i in range(T):
            if not hit[i]:
                assert torch.isfinite(out[:, :, i]).all(), (which, i)
                # (As before but for the order of a few sums: 32 of a float32 sum's half steps, 8 of the others'.)
                most = 4 * torch.finfo(dtype).eps * clean[:, :, i].abs().max()
                assert (out[:, :, i].float() - clean[:, :, i].float()).abs().max() <= most, (which, i)
            elif which == "v" and not c.narrow:
                assert (out[0, :, i, 7] == value).all() if value == value else torch.isnan(out[0, :, i, 7]).all()
                assert torch.isfinite(out[0, :, i, :7]).all() and torch.isfinite(out[0, :, i, 8:]).all()
            elif which != "k" or value != value or c.narrow:  # (a key's infinity may be a score of -infinity)
                assert not torch.isfinite(out[0, :, i]).all(), (which, i)


def test_counts_positions_and_pages(gpu_device):
    T = 10
    for dtype, kv in ((BF, BF), (F32, I8)):
        c = Cache(gpu_device, 8, 2, 64, 16, 4, dtype, kv)
        c.table[3, 1], c.table[4, 3] = -1, c.P
        pos = [20, 0, -1, 40, 45, 58, 64, 2 ** 40]
        parents = [tree(T, b) for b in range(8)]
        step(c, pos, parents)
        step(c, pos, parents, counts=[3, 0, 5, 10, 99, -4, 1, 2])
        step(c, [-5, -2 ** 40, 10, 64, 65, 0, 0, 0], parents, G=3, counts=[9, 9, 1, 4, 4, 10, 2 ** 40, -2 ** 40])
        step(c, pos, parents, window=5, sinks=3)


def test_no_table_and_no_sequences(gpu_device):
    c = Cache(gpu_device, 2, 2, 32, 16, 2, BF)
    c.table = c.table[:, :0]
    step(c, [0, 3], [tree(4, 0)] * 2)
    z = torch.zeros(0, 2, 3, 32, dtype=BF, device=gpu_device)
    out = paged_tree_step(z, z, z, c.k, c.v, c.table[:0], torch.zeros(0, dtype=torch.int64, device=gpu_device))
    assert out.shape == (0, 2, 3, 32)


@pytest.mark.parametrize("layout", ["tokens", "plain", "unaligned"])
@pytest.mark.parametrize("pool", ["heads", "tokens", "wide"])
@pytest.mark.parametrize("kv", [BF, E4])
def test_layouts(gpu_device, layout, pool, kv):
    pos = [61, 18]
    c = Cache(gpu_device, 2, 3, 64, 16, 6, BF, kv, [p + 20 for p in pos], layout=pool)
    step(c, pos, [tree(20, b) for b in range(2)], 2, layout=layout)


def test_odd_scales(gpu_device):
    """Scale bytes at odd places, one after another or not: the same results and bytes."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, h, 9, 64, generator=g).to(gpu_device, F16) for h in (6, 3, 3))
    pos = torch.tensor([40, 7], device=gpu_device)
    for kv in (E4, I8):
        a, b = (Cache(gpu_device, 2, 3, 64, 16, 5, F16, kv) for _ in range(2))
        for n in ("k_scale", "v_scale"):
            wide = torch.zeros(b.P, 3, 33, dtype=torch.uint8, device=gpu_device)
            view = wide[..., 1::2] if n == "k_scale" else wide[..., 1:17]
            view.copy_(getattr(b, n).view(torch.uint8))
            setattr(b, n, view.view(torch.float8_e8m0fnu))
        x = paged_tree_step(q, k, v, a.k, a.v, a.table, pos, **a.state)
        y = paged_tree_step(q, k, v, b.k, b.v, b.table, pos, **b.state)
        assert torch.equal(x, y) and torch.isfinite(x).all()
        same(a.k, b.k)
        for n in ("k_scale", "v_scale"):
            assert torch.equal(getattr(a, n).view(torch.uint8), getattr(b, n).view(torch.uint8))


@pytest.mark.parametrize("dtype,kv,D,G,T", [(BF, BF, 64, 1, 26), (BF, E4, 128, 4, 64), (F16, I8, 80, 5, 3), (F32, F32, 32, 1, 7),
                                            (F32, E4, 96, 2, 33), (BF, BF, 128, 8, 1), (F16, F16, 128, 2, 64), (F32, F32, 128, 1, 64)])
def test_long(gpu_device, dtype, kv, D, G, T):
    """Caches that are split over workgroups: ragged ones, and with a window whose tiles begin anywhere."""
    pos = [2000, 1, 777, 1503]
    c = Cache(gpu_device, 4, 2, D, 64, 33, dtype, kv, [p + T for p in pos])
    junk(c, pos)
    for kw in (dict(), dict(window=700, sinks=33)):
        a = step(c, pos, [tree(T, b) for b in range(4)], G, **kw)
        assert torch.equal(a, step(c, pos, [tree(T, b) for b in range(4)], G, **kw))  # the same bits again


def test_stored_rows_and_scales_of_scores(gpu_device):
    """Without new rows the draft is attended as the pages hold it; negative, zero and sharp softmax scales."""
    for dtype, kv in ((BF, BF), (F32, F32), (F16, E4)):
        c = Cache(gpu_device, 2, 2, 64, 16, 6, dtype, kv)
        for scale in (None, 0.0, -0.7, 30.0):
            step(c, [60, 11], [tree(17, b) for b in range(2)], 2, fresh=False, scale=scale)
            step(c, [60, 11], [tree(17, b) for b in range(2)], 1, scale=scale)


def test_chain_is_steps(gpu_device):
    """A chain of tokens attends what as many single-token steps attend, and leaves the same cache."""
    for dtype, kv in ((F32, F32), (BF, E4)):
        a = Cache(gpu_device, 3, 2, 64, 16, 6, dtype, kv, seed=5)
        b = Cache(gpu_device, 3, 2, 64, 16, 6, dtype, kv, seed=5)
        g = torch.Generator().manual_seed(0)
        q, k, v = (torch.randn(3, h, 6, 64, generator=g).to(gpu_device, dtype) for h in (4, 2, 2))
        pos = torch.tensor([15, 0, 70], device=gpu_device)
        out = paged_tree_step(q, k, v, a.k, a.v, a.table, pos, **a.state)
        for i in range(6):
            one = paged_decode_step(q[:, :, i], k[:, :, i], v[:, :, i], b.k, b.v, b.table, pos + i, **b.state)
            tol = 2.0 ** -18 if dtype == F32 else 2.0 ** -6
            assert (out[:, :, i] - one).abs().max() <= tol * 4
        same(a.k, b.k)
        same(a.v, b.v)


@pytest.mark.parametrize("kv", [None, E4, I8])
def test_draft_accept_and_go_on(gpu_device, kv):
    """PagedKVCache: prompts, a draft, its accepted rows, another draft, a single-token step: at the end the cache holds
    what writing the accepted rows one by one leaves, and each draft attends that."""
    B, H, G, D, T = 3, 2, 2, 64, 9
    g = torch.Generator().manual_seed(2)
    cache = PagedKVCache(B, H, D, 200, BF, gpu_device, kv_dtype=kv, page_size=16)
    plain = PagedKVCache(B, H, D, 200, BF, gpu_device, kv_dtype=kv, page_size=16)

    def randn(*s):
        return torch.randn(*s, generator=g).to(gpu_device, BF)

    k, v = randn(B, H, 40, D), randn(B, H, 40, D)
    counts = torch.tensor([40, 7, 21], device=gpu_device)
    for c in (cache, plain):
        c.prefill(k, v, counts)
    cache.pos[1] = plain.pos[1] = -1  # out of use
    for r in range(4):
        parents = torch.tensor([tree(T, r * 3 + b) for b in range(B)], device=gpu_device)
        tokens = torch.randint(0, 4, (B, T), generator=g).to(gpu_device)
        q, k, v = randn(B, H * G, T, D), randn(B, H, T, D), randn(B, H, T, D)
        out = cache.tree_step(q, k, v, parents)
        assert (out[1] == 0).all()
        rk, rv = (t.cpu().double() for t in cache.read())
        before = cache.pos.tolist()
        for b in (0, 2):
            nodes = po.tree_rows(parents[b].tolist(), T)
            kk, vv = (torch.stack([po_rows(t[b:b + 1], kv)[0] for t in (x,)])[0] for x in (k, v))
            for i, nd in enumerate(nodes):
                sees = nd[0]
                ks = torch.cat([rk[b, :, :before[b]], kk[:, sees]], 1)
                vs = torch.cat([rv[b, :, :before[b]], vv[:, sees]], 1)
                ref, mass, size = po.attend(q[b, :, i].cpu(), ks, vs, D ** -0.5)
                assert ((out[b, :, i].double().cpu() - ref).abs() <=
                        po.tree_bound(ref, mass, size, D, ks.shape[1], BF, kv or BF, T * G)).all()
        picks = torch.randint(0, 4, (B, T), generator=g).to(gpu_device)
        path, n, _ = draft_tree_accept(tokens, parents, picks)
        cache.accept(k, v, path, n)
        for b in range(B):
            for i in range(int(n[b])):
                one = torch.zeros(B, dtype=torch.int64, device=gpu_device)
                one[b] = 1
                j = int(path[b, i])
                plain.write(k[:, :, j:j + 1], v[:, :, j:j + 1], one)
        assert cache.pos.tolist() == plain.pos.tolist() == [before[b] + (int(n[b]) if b != 1 else 0) for b in range(B)]
        for x, y in zip(cache.read(), plain.read()):
            assert torch.equal(x, y)
    q, k, v = randn(B, H * G, D), randn(B, H, D), randn(B, H, D)
    assert torch.equal(cache.step(q, k, v), plain.step(q, k, v))


def po_rows(t, kv):
    """Rows [1,H,T,D] as a cache keeps them, float64."""
    x = t[0].cpu()
    if kv is None:
        return x.double()[None]
    codes, e = po.encode(x, kv)
    return (codes * (2.0 ** (e.double() - 127))[..., None])[None]


def test_graphs(gpu_device):
    """Two captured steps share the pool of workspaces; replays between eager calls give the eager results."""
    dev, T = gpu_device, 20
    for dtype, kv in ((BF, BF), (F32, E4)):
        a = Cache(dev, 3, 2, 64, 64, 40, dtype, kv, seed=1)
        b = Cache(dev, 3, 2, 64, 64, 40, dtype, kv, seed=1)
        pos = torch.tensor([2000, 5, 900], device=dev)
        parents = torch.tensor([tree(T, i) for i in range(3)], device=dev)
        g = torch.Generator().manual_seed(0)
        q, k, v = (torch.randn(3, h, T, 64, generator=g).to(dev, dtype) for h in (4, 2, 2))

        def call(c, w):
            return paged_tree_step(q, k, v, c.k, c.v, c.table, pos, parents, window=w, sinks=3, **c.state)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(a, None), call(a, 600)
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for w in (None, 600):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
                out = call(a, w)
            graphs.append((graph, out, w))
        for r in range(3):
            pos += r
            q.mul_(-1)
            parents.copy_(torch.tensor([tree(T, i + r) for i in range(3)], device=dev))
            for graph, out, w in graphs:
                graph.replay()
                got = out.clone()
                want = call(b, w)
                torch.cuda.synchronize()
                assert torch.equal(got, want)
                same(a.k, b.k)


def test_other_streams_and_traced(gpu_device):
    c = Cache(gpu_device, 2, 2, 64, 16, 6, BF)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, h, 5, 64, generator=g).to(gpu_device, BF) for h in (4, 2, 2))
    pos = torch.tensor([30, 4], device=gpu_device)
    pt = torch.tensor(tree(5, 0), device=gpu_device)
    want = paged_tree_step(q, k, v, c.k, c.v, c.table, pos, pt, window=9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_tree_step(q, k, v, c.k, c.v, c.table, pos, pt, window=9)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    f = torch.compile(lambda *a: paged_tree_step(*a, window=9) * 1.0, backend="eager")
    assert torch.equal(f(q, k, v, c.k, c.v, c.table, pos, pt), want)
    version = c.k._version
    paged_tree_step(q, k, v, c.k, c.v, c.table, pos, pt)
    assert c.k._version > version
    version = c.k._version
    paged_tree_step(q, None, None, c.k, c.v, c.table, pos, pt)
    assert c.k._version == version


@pytest.mark.parametrize("kv", [E4, I8])
@pytest.mark.parametrize("D", [32, 128])
def test_float16_over_8_bits(gpu_device, kv, D):
    """Float16 queries over 8-bit rows: 20 nodes give what 16 of them give, whose weights are two bfloat16 terms.  Both are
    within 2^-16 of the weights' mass, at most the largest value, and half a step of the output (2^-11 of it) of the exact
    result, so within 2^-15 max|v| and 2^-10 |x| of each other.  (One term would be off by up to 2^-9 of the mass.)"""
    pos, G = [300, 45], 1
    outs = []
    for T in (20, 16):
        c = Cache(gpu_device, 2, 2, D, 16, 24, F16, kv, [p + 20 for p in pos])
        junk(c, pos)
        g = torch.Generator().manual_seed(9)
        q, k, v = (torch.randn(2, 2 * n, 20, D, generator=g).to(gpu_device, F16)[:, :, :T] for n in (G, 1, 1))
        outs.append(paged_tree_step(q, k, v, c.k, c.v, c.table, torch.tensor(pos, device=gpu_device), **c.state).double().cpu()[:, :, :16])
        largest = max(torch.nan_to_num(c.rows("v", b, pos[b] + 16)).abs().max().item() for b in range(2))
    x, y = outs
    assert torch.isfinite(x).all() and ((x - y).abs() <= 2.0 ** -10 * y.abs() + 2.0 ** -15 * largest).all()
