"""Drafted-token steps on the GPU at the ends of their range: huge scores, NaN codes of 8-bit pages, parents past 32
bits, pools beyond the caches."""

import pytest
import torch

from dwarf_amd import draft_tree_accept, paged_tree_step
from oracle import paged_oracle as po
from tests.test_paged_gpu import Cache
from tests.test_paged_tree_gpu import BF, E4, F16, F32, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,kv", [(F16, F16), (F16, E4), (BF, BF), (F32, F32)])
@pytest.mark.parametrize("T", [8, 30])
@pytest.mark.parametrize("power", [14, 20, 22, 23, 24, 25, 26, 28])
def test_huge_scores(gpu_device, dtype, kv, T, power):
    """Scores up to 2^40 give the row of the largest.  Sums of |q||k| are below 2^12, so that a score is off by 40 2^-12 times
    the scale at most, and one that is ahead by 2^8 besides leaves the others exp(-2^8) of its weight: nothing.  What is left of
    the row is its weight's two 16-bit terms, 2^-16 of it, or one that is exact, and a half step of the output."""
    D, pos = 32, [200, 31, 0, 77]
    c = Cache(gpu_device, 4, 1, D, 16, 16, dtype, kv, [p + T for p in pos])
    g = torch.Generator().manual_seed(power)
    q, k, v = (torch.randn(4, 1, T, D, generator=g).to(dtype).to(gpu_device) for _ in range(3))
    parents = [tree(T, b) for b in range(4)]
    out = paged_tree_step(q, k, v, c.k, c.v, c.table, torch.tensor(pos, device=gpu_device), torch.tensor(parents, device=gpu_device),
                          softmax_scale=2.0 ** power, **c.state).double().cpu()
    sure = 0
    for b, n in enumerate(pos):
        nodes = po.tree_rows(parents[b], T)
        kk, vv = c.rows("k", b, n + T)[0], c.rows("v", b, n + T)[0]
        for i, node in enumerate(nodes):
            sees = po.tree_sees(node, nodes, n)
            x = q[b, 0, i].double().cpu()
            assert torch.isfinite(out[b, 0, i]).all(), (b, i)
            assert (kk[sees].abs() @ x.abs()).max() < 2 ** 12
            s = torch.cat([kk[sees] @ x, torch.tensor([-torch.inf], dtype=torch.float64)])
            first, second = s.topk(2).values.tolist()
            if first - second > 2 * 40 * 2.0 ** -12 + 2.0 ** (8 - power):
                sure += 1
                want = vv[sees[int(s.argmax())]]
                assert ((out[b, 0, i] - want).abs() <= want.abs() * (2.0 ** -16 + torch.finfo(dtype).eps / 2)).all(), (b, i)
    assert sure > 3 * T


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("T,G", [(12, 1), (30, 1), (50, 2)])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_nan_codes_stay_with_who_sees_them(gpu_device, dtype, D, T, G, code):
    """Pages from elsewhere may hold e4m3's NaN under an ordinary scale: the nodes that see its row get NaN in that element, and
    everything else is what it was, bit by bit (a hidden row's weight is 0 and its value no part of the sums)."""
    n, parents = 75, tree(T, 4)
    nodes = po.tree_rows(parents, T)
    c = Cache(gpu_device, 1, 2, D, 16, 9, dtype, E4, [n + T])
    q = torch.randn(1, 2 * G, T, D, generator=torch.Generator().manual_seed(1)).to(dtype).to(gpu_device)
    pt, pos = torch.tensor(parents, device=gpu_device), torch.tensor([n], device=gpu_device)

    def call(**kw):
        return paged_tree_step(q, None, None, c.k, c.v, c.table, pos, pt, **kw, **c.state).cpu()

    for at, kw in ((n + 3, {}), (n + T - 1, {}), (n - 9, dict(window=12, sinks=2)), (3, dict(window=40, sinks=5)), (n + 2, dict(window=3))):
        hit = torch.tensor([at in po.tree_sees(node, nodes, n, kw.get("window"), kw.get("sinks", 0)) for node in nodes])
        want = call(**kw)
        assert torch.isfinite(want).all()
        cell = c.v.view(torch.uint8)[int(c.table[0, at // 16]), 1, at % 16]
        old = cell.clone()
        cell[7] = cell[D - 1] = code
        got = call(**kw)
        cell.copy_(old)
        want[:, G:, hit, 7] = want[:, G:, hit, D - 1] = torch.nan
        assert torch.equal(torch.isnan(got), torch.isnan(want)), (at, kw)
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0)), (at, kw)
        assert not hit.all() or at == 3
        # A key's scores are NaN, and so all of such a node's output.
        cell = c.k.view(torch.uint8)[int(c.table[0, at // 16]), 1, at % 16]
        old = cell.clone()
        cell[5] = code
        got = call(**kw)
        cell.copy_(old)
        want[:, G:, hit] = torch.nan
        assert torch.equal(torch.isnan(got), torch.isnan(want)), (at, kw)
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0)), (at, kw)


@pytest.mark.parametrize("shared", [True, False])
def test_parents_past_32_bits(gpu_device, shared):
    """64-bit parents that 32 bits would make a node of: such nodes, and those below them, are none."""
    T, wrong = 12, [2 ** 32, 2 ** 32 - 1, -2 ** 32 - 1, 2 ** 40 + 1, -2 ** 63, 2 ** 63 - 1]
    parents = tree(T, 2)
    for i, w in zip((1, 3, 5, 6, 8, 11), wrong):
        parents[i] = w
    small = [p if -1 <= p < T else -2 for p in parents]
    assert sum(x is None for x in po.tree_rows(parents, T)) >= 6
    c = Cache(gpu_device, 2, 1, 64, 16, 6, BF, lengths=[40 + T, 5 + T])
    q, k, v = (torch.randn(2, 1, T, 64, generator=torch.Generator().manual_seed(i)).to(BF).to(gpu_device) for i in range(3))
    pos = torch.tensor([40, 5], device=gpu_device)
    tokens = torch.zeros(2, T, dtype=torch.int64, device=gpu_device)

    def table(p, dtype):
        return torch.tensor(p if shared else [p, p], dtype=dtype).to(gpu_device)

    want = paged_tree_step(q, k, v, c.k, c.v, c.table, pos, table(small, torch.int32))
    for i, node in enumerate(po.tree_rows(parents, T)):
        assert (want[:, :, i] == 0).all() == (node is None)
    assert torch.equal(paged_tree_step(q, k, v, c.k, c.v, c.table, pos, table(parents, torch.int64)), want)
    for a, b in zip(draft_tree_accept(tokens, table(parents, torch.int64), tokens), draft_tree_accept(tokens, table(small, torch.int32), tokens)):
        assert torch.equal(a, b)
    # Unsigned ones: -1 is their largest number, no node.
    line = [0, 0, 1, 2 ** 32 - 1, 2, 2 ** 32 - 2]
    for dtype, more in ((torch.uint32, 0), (torch.uint64, 2 ** 64 - 2 ** 32)):
        big = [x + more if x > 99 else x for x in line]
        p = table(big + [0] * (T - 6), torch.uint64).to(dtype)
        path, n, _ = draft_tree_accept(tokens, p, tokens)
        assert path[:, :4].tolist() == [[0, 1, 2, 4]] * 2 and n.tolist() == [4, 4]
        assert (paged_tree_step(q, k, v, c.k, c.v, c.table, pos, p) == 0).all()


@pytest.mark.parametrize("dtype,kv", [(BF, BF), (F16, E4), (F32, F32)])
@pytest.mark.parametrize("T", [1, 13])
def test_pools_beyond_the_caches(gpu_device, dtype, kv, T):
    """Rows of pools above 85 MiB are read past the caches' retention: the same bits as from a small pool."""
    D, page, pos = 64, 64, [500, 77, 260]
    c = Cache(gpu_device, 3, 2, D, page, 10, dtype, kv, [p + T for p in pos])
    P = (86 << 20) // (2 * 2 * page * D * kv.itemsize) + 1  # (two pools of two heads)
    at = torch.randperm(P, generator=torch.Generator().manual_seed(3))[:c.P].to(gpu_device)
    big = {}
    for n in ("k", "v", "k_scale", "v_scale"):
        x = getattr(c, n)
        if x is not None:
            as_bytes = (lambda t: t.view(torch.uint8)) if x.element_size() == 1 else (lambda t: t)
            big[n] = torch.zeros(P, *x.shape[1:], dtype=as_bytes(x).dtype, device=gpu_device)
            big[n][at] = as_bytes(x)
            big[n] = big[n].view(x.dtype)
    inside = (c.table >= 0) & (c.table < c.P)
    table = torch.where(inside, at[c.table.clamp(0, c.P - 1).long()].int(), -1)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(3, h, T, D, generator=g).to(dtype).to(gpu_device) for h in (4, 2, 2))
    p, pt = torch.tensor(pos, device=gpu_device), torch.tensor([tree(T, b) for b in range(3)], device=gpu_device)
    for kw in ({}, dict(window=100, sinks=3)):
        want = paged_tree_step(q, k, v, c.k, c.v, c.table, p, pt, **kw, **c.state)
        got = paged_tree_step(q, k, v, big["k"], big["v"], table, p, pt, **kw, k_scale=big.get("k_scale"), v_scale=big.get("v_scale"))
        assert torch.equal(got, want) and torch.isfinite(got).all()
        for n in big:
            a, b = (t.view(torch.uint8) if t.element_size() == 1 else t for t in (big[n], getattr(c, n)))
            assert torch.equal(a[at], b)
