"""Sampling and the walk over drafted tokens without a GPU: the oracle against torch, the refusals of the public
functions, and the C ABI's argument checks."""

import ctypes
import math

import pytest
import torch

import dwarf_amd
from dwarf_amd import _lib, draft_tree_accept, paged_kv_write, sample_tokens
from oracle import sample_oracle as so


def test_oracle_draws_the_distribution():
    """Over a grid of u each token of the kept set comes up in proportion to its probability."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, generator=g).double()
    p = torch.softmax(x / 0.7, 0)
    order = torch.argsort(x, descending=True)
    before = torch.cumsum(p[order], 0) - p[order]
    kept = order[before <= 0.8]
    q = torch.zeros(40, dtype=torch.float64)
    q[kept] = p[kept] / p[kept].sum()
    n = 4000
    draws = torch.tensor([so.sample(x.tolist(), (i + 0.5) / n, 0.7, top_p=0.8)[0] for i in range(n)])
    # A token's share of the grid differs from its probability by less than two points.
    assert (torch.bincount(draws, minlength=40).double() / n - q).abs().max() <= 2.0 / n
    token, logp, _ = so.sample(x.tolist(), 0.3, 0.7, top_p=0.8)
    assert abs(logp - math.log(q[token])) < 1e-12


def test_oracle_limits():
    row = [1.0, 3.0, 3.0, 2.0, -math.inf, math.nan]
    assert so.sample(row, 0.99, top_k=1)[0] == 1 and so.sample(row, 0.99, top_k=2)[0] == 2
    assert so.sample(row, 0.0, top_p=0.0)[0] == 1
    assert so.sample(row, 0.999)[0] == 3 and so.sample(row, 0.999, min_p=0.5)[0] == 2
    assert so.sample(row, 0.5, temperature=0.0)[:2] == (1, 0.0)
    assert so.sample([-math.inf, math.nan], 0.5)[:2] == (-1, -math.inf)
    assert so.sample([0.0, math.inf, 5.0, math.inf], 0.6)[:2] == (3, -math.log(2))


def test_oracle_walk():
    parents, tokens = [-1, 0, 0, 1, 2, 3], [5, 7, 8, 9, 9, 4]
    assert so.walk(tokens, parents, [8, 0, 9, 0, 2, 0]) == ([0, 2, 4], 2)
    assert so.walk(tokens, parents, [7, 9, 0, 4, 0, 1]) == ([0, 1, 3, 5], 1)
    assert so.walk(tokens, parents, [7, 9, 0, 4, 0, 1], 3) == ([0, 1], 9)
    assert so.walk(tokens, parents, [6, 0, 0, 0, 0, 0]) == ([0], 6) and so.walk(tokens, parents, [0] * 6, 0) == ([], -1)


@pytest.mark.parametrize("case", [
    lambda: sample_tokens(torch.zeros(2, 0), torch.rand(2)),
    lambda: sample_tokens(torch.zeros(()), torch.rand(())),
    lambda: sample_tokens(torch.zeros(2, 4, dtype=torch.float64), torch.rand(2)),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(3)),
    lambda: sample_tokens(torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64)),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), -0.1),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), math.nan),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), top_k=-1),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), top_p=1.1),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), top_p=math.nan),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), min_p=-0.5),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), torch.ones(3)),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), top_k=torch.ones(2)),
    lambda: sample_tokens(torch.zeros(2, 4), torch.rand(2), top_p=torch.ones(2, dtype=torch.int64)),
    lambda: draft_tree_accept(torch.zeros(2, 65, dtype=torch.int64), torch.zeros(65, dtype=torch.int32),
                              torch.zeros(2, 65, dtype=torch.int64)),
    lambda: draft_tree_accept(torch.zeros(2, 0, dtype=torch.int64), torch.zeros(0, dtype=torch.int32),
                              torch.zeros(2, 0, dtype=torch.int64)),
    lambda: draft_tree_accept(torch.zeros(2, 4), torch.zeros(4, dtype=torch.int32), torch.zeros(2, 4)),
    lambda: draft_tree_accept(torch.zeros(2, 4, dtype=torch.int64), torch.zeros(3, dtype=torch.int32),
                              torch.zeros(2, 4, dtype=torch.int64)),
    lambda: draft_tree_accept(torch.zeros(2, 4, dtype=torch.int64), torch.zeros(4, dtype=torch.int32),
                              torch.zeros(2, 3, dtype=torch.int64)),
    lambda: draft_tree_accept(torch.zeros(2, 4, dtype=torch.int64), torch.zeros(4, dtype=torch.int32),
                              torch.zeros(2, 4, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)),
])
def test_refused(case):
    with pytest.raises(AssertionError):
        case()


def test_refused_gradients_and_devices():
    with pytest.raises(RuntimeError, match="gradient"):
        sample_tokens(torch.zeros(2, 4, requires_grad=True), torch.rand(2), return_logprobs=True)
    with pytest.raises(RuntimeError, match="GPU"):
        sample_tokens(torch.zeros(2, 4, requires_grad=True), torch.rand(2))
    z = torch.zeros(2, 4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        draft_tree_accept(z, z, z)


def test_write_refuses_rows():
    pages = torch.zeros(4, 2, 16, 32)
    k, table, pos = torch.zeros(2, 2, 3, 32), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    for rows in (torch.zeros(2, 3), torch.zeros(3, 3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)):
        with pytest.raises(AssertionError, match="rows must be"):
            paged_kv_write(k, k, pages, pages.clone(), table, pos, rows=rows)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_kv_write(k, k, pages, pages.clone(), table, pos, rows=torch.zeros(2, 5, dtype=torch.int64))


def _sample_args(**kw):
    a = _lib.SampleArgs()
    a.B, a.V, a.dtype, a.temperature, a.top_p = 2, 10, _lib.DSQG_F32, 1.0, 1.0
    a.logits = a.u = a.tokens = 0x10000
    a.logits_stride = 10
    for n, x in kw.items():
        setattr(a, n, x)
    return a


def test_abi_refuses_bad_sampling():
    lib = _lib.load()

    def call(**kw):
        return lib.dsqg_sample(ctypes.byref(_sample_args(**kw)), None)

    assert lib.dsqg_sample(None, None) == _lib.DSQG_EINVAL
    assert call(B=0) == _lib.DSQG_OK
    for bad in (dict(B=-1), dict(V=0), dict(dtype=3), dict(dtype=-1), dict(logits=None), dict(u=None), dict(tokens=None),
                dict(logits=0x10002), dict(logits_stride=-1), dict(logits_stride=1 << 51), dict(u_is_double=2),
                dict(temperature=math.nan), dict(top_p=math.nan), dict(min_p=math.nan)):
        assert call(**bad) == _lib.DSQG_EINVAL, bad
    assert call(V=(1 << 30) + 1) == _lib.DSQG_EUNSUPPORTED


def test_abi_refuses_bad_trees():
    lib = _lib.load()

    def call(**kw):
        a = _lib.TreeAcceptArgs()
        a.B, a.T = 2, 5
        a.tokens = a.parents = a.picks = a.path = a.n = a.next = 0x10000
        a.tokens_stride = a.parents_stride = a.picks_stride = 5
        for n, x in kw.items():
            setattr(a, n, x)
        return lib.dsqg_tree_accept(ctypes.byref(a), None)

    assert lib.dsqg_tree_accept(None, None) == _lib.DSQG_EINVAL
    assert call(B=0) == _lib.DSQG_OK and call(T=65) == _lib.DSQG_EUNSUPPORTED
    for bad in (dict(B=-1), dict(T=0), dict(tokens=None), dict(parents=None), dict(picks=None), dict(path=None), dict(n=None),
                dict(next=None), dict(tokens_stride=-1), dict(parents_stride=1 << 51)):
        assert call(**bad) == _lib.DSQG_EINVAL, bad


def test_traced_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 3, 100, dtype=torch.bfloat16, device="cuda")
        u = torch.empty(2, 3, device="cuda")
        t = dwarf_amd.sample_tokens(x, u, 0.8, top_k=u.long(), top_p=u)
        assert t.shape == (2, 3) and t.dtype == torch.int64
        t, lp = dwarf_amd.sample_tokens(x, u, u, return_logprobs=True)
        assert lp.shape == (2, 3) and lp.dtype == torch.float32
        z = torch.empty(2, 7, dtype=torch.int64, device="cuda")
        path, n, nxt = dwarf_amd.draft_tree_accept(z, z, z)
        assert path.shape == (2, 7) and n.shape == nxt.shape == (2,)


def test_structs_match_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    header = Path(__file__).resolve().parents[1] / "include" / "dsqg.h"
    probes = {"dsqg_sample_args": _lib.SampleArgs, "dsqg_tree_accept_args": _lib.TreeAcceptArgs,
              "dsqg_paged_write_args": _lib.PagedWriteArgs}
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    for c, cls in probes.items():
        src.append(f'printf("%zu\\n", sizeof({c}));')
        src += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "p.c").write_text("\n".join(src + ["return 0;}"]))
    subprocess.run([shutil.which("gcc") or "cc", str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    out = [int(x) for x in subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for cls in probes.values():
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert out == want
