"""Steps of drafted tokens without a GPU: the oracle, the refusals of the public function and the C ABI's checks."""

import ctypes

import pytest
import torch

from dwarf_amd import _lib, paged_tree_step
from oracle import paged_oracle as po

BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def test_oracle_trees():
    nodes = po.tree_rows([-1, 0, 1, 0, 3, 7, -2, -1, 5], 9)
    assert nodes[2] == ([0, 1, 2], 2) and nodes[4] == ([0, 3, 4], 2) and nodes[7] == ([7], 0)
    assert nodes[5] is None and nodes[6] is None and nodes[8] is None
    assert po.tree_rows([-1, 0, 1], 2)[2] is None
    assert po.tree_sees(nodes[4], nodes, 3) == [0, 1, 2, 3, 6, 7]
    assert po.tree_sees(nodes[4], nodes, 10, 3, 0) == [10, 13, 14]
    assert po.tree_sees(nodes[4], nodes, 10, 4, 1) == [0, 9, 10, 13, 14]
    assert po.tree_sees(nodes[4], nodes, 2, 1, 3) == [0, 1, 2, 6]


def _args(B=2, H=2, G=2, T=5, D=32, dtype=BF, kv=BF):
    pages = torch.zeros(6, H, 16, D, dtype=kv)
    a = dict(q=torch.zeros(B, H * G, T, D, dtype=dtype), k_new=torch.zeros(B, H, T, D, dtype=dtype),
             v_new=torch.zeros(B, H, T, D, dtype=dtype), k_pages=pages, v_pages=pages.clone(),
             page_table=torch.zeros(B, 3, dtype=torch.int32), pos=torch.zeros(B, dtype=torch.int64),
             parents=torch.zeros(T, dtype=torch.int32))
    if kv.itemsize == 1:
        a["k_scale"] = torch.zeros(6, H, 16, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        a["v_scale"] = a["k_scale"].clone()
    return a


def test_only_the_gpu_is_missing():
    for dtype, kv in ((BF, BF), (torch.float16, E4)):
        with pytest.raises(RuntimeError, match="GPU"):
            paged_tree_step(**_args(dtype=dtype, kv=kv))
        with pytest.raises(RuntimeError, match="GPU"):
            paged_tree_step(**dict(_args(dtype=dtype, kv=kv), parents=None, k_new=None, v_new=None))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 4, 32, dtype=BF)), dict(q=torch.zeros(2, 3, 5, 32, dtype=BF)), dict(q=torch.zeros(3, 4, 5, 32, dtype=BF)),
    dict(q=torch.zeros(2, 4, 5, 64, dtype=BF)), dict(q=torch.zeros(2, 4, 5, 32)), dict(q=torch.zeros(2, 4, 4, 32, dtype=BF)),
    dict(k_new=None), dict(v_new=None), dict(k_new=torch.zeros(2, 2, 4, 32, dtype=BF)), dict(v_new=torch.zeros(2, 2, 5, 32)),
    dict(parents=torch.zeros(4, dtype=torch.int32)), dict(parents=torch.zeros(5)), dict(parents=torch.zeros(3, 5, dtype=torch.int32)),
    dict(counts=torch.zeros(3, dtype=torch.int64)), dict(counts=torch.zeros(2)), dict(window=0), dict(window=-3), dict(sinks=-1),
    dict(k_scale=torch.zeros(6, 2, 16, dtype=torch.uint8).view(torch.float8_e8m0fnu)),
    dict(parents=None, counts=torch.zeros(2, 1, dtype=torch.int64)),
])
def test_refused(change):
    with pytest.raises(AssertionError):
        paged_tree_step(**dict(_args(), **change))


def test_refuses_sizes_and_gradients():
    for T in (65, 0):
        with pytest.raises(AssertionError, match="64"):
            paged_tree_step(**_args(T=T))
    a = _args(dtype=torch.float32, kv=torch.float32)
    a["q"].requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        paged_tree_step(**a)


def _abi(**kw):
    a = _lib.PagedTreeArgs()
    c = a.cache
    c.dtype = c.cache_dtype = _lib.DSQG_BF16
    c.B, c.Hkv, c.D, c.P, c.page, c.M = 2, 2, 64, 6, 16, 3
    c.k_pages = c.v_pages = c.page_table = 0x10000
    for s in (c.k_stride, c.v_stride):
        s[0], s[1], s[2] = 2 * 16 * 64, 16 * 64, 64
    c.table_stride = 3
    a.H, a.T = 4, 5
    a.q = a.k_new = a.v_new = a.parents = a.pos = a.out = 0x10000
    for s in (a.q_stride, a.k_new_stride, a.v_new_stride):
        s[0], s[1], s[2] = 4 * 5 * 64, 5 * 64, 64
    a.parents_stride = 5
    a.workspace, a.workspace_bytes = 0x10000, 1 << 30
    for n, x in kw.items():
        (setattr(c, n[2:], x) if n.startswith("c_") else setattr(a, n, x))
    return a


def test_abi_checks():
    lib = _lib.load()

    def call(**kw):
        return lib.dsqg_paged_tree(ctypes.byref(_abi(**kw)), None)

    assert lib.dsqg_paged_tree(None, None) == _lib.DSQG_EINVAL
    assert call(c_B=0) == _lib.DSQG_OK
    for bad in (dict(H=3), dict(H=0), dict(H=-4), dict(T=0), dict(window=-1), dict(sinks=-1), dict(q=None), dict(q=0x10008),
                dict(pos=None), dict(out=None), dict(out=0x10004), dict(k_new=None), dict(v_new=None), dict(k_new=0x10002),
                dict(parents_stride=-1), dict(c_cache_dtype=_lib.DSQG_F32), dict(c_P=0), dict(c_page=24), dict(c_page_table=None)):
        assert call(**bad) == _lib.DSQG_EINVAL, bad
    for bad in (dict(T=65), dict(c_D=48), dict(c_page=8), dict(c_M=1 << 27)):
        assert call(**bad) == _lib.DSQG_EUNSUPPORTED, bad
    n = ctypes.c_size_t(7)
    assert lib.dsqg_paged_tree_workspace_size(ctypes.byref(_abi()), None) == _lib.DSQG_EINVAL
    assert lib.dsqg_paged_tree_workspace_size(ctypes.byref(_abi(c_M=4096)), ctypes.byref(n)) == _lib.DSQG_OK and n.value > 0
    assert call(c_M=4096, workspace=None) == _lib.DSQG_EWORKSPACE
    assert call(c_M=4096, workspace_bytes=n.value - 1) == _lib.DSQG_EWORKSPACE
    assert call(c_M=4096, workspace=0x10010) == _lib.DSQG_EINVAL


def test_traced_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        a = {n: t.to("cuda") for n, t in _args().items()}
        out = paged_tree_step(**a, window=4)
        assert out.shape == (2, 4, 5, 32) and out.stride() == (5 * 4 * 32, 32, 4 * 32, 1)


def test_struct_matches_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    header = Path(__file__).resolve().parents[1] / "include" / "dsqg.h"
    cls = _lib.PagedTreeArgs
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){",
           'printf("%zu\\n", sizeof(dsqg_paged_tree_args));']
    src += [f'printf("%zu\\n", offsetof(dsqg_paged_tree_args, {f}));' for f, _ in cls._fields_]
    (tmp_path / "p.c").write_text("\n".join(src + ["return 0;}"]))
    subprocess.run([shutil.which("gcc") or "cc", str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
