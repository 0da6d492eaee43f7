"""Sizes past what grids hold are refused as such before anything is launched (no GPU is needed, and none is used)."""

import ctypes

import pytest
import torch

from dwarf_amd import _lib, ops
from tests.test_paged_tree_cpu import _abi
from tests.test_window_cpu import _fill, _shape


def _window(shape):
    """Statuses of the forward, the size query and the backward."""
    lib, n = _lib.load(), ctypes.c_size_t(0)
    f, b = _lib.WindowFwdArgs(), _lib.WindowBwdArgs()
    f.shape = b.shape = shape
    _fill(f, ("q", "k", "v", "out"))
    _fill(b, ("q", "k", "v", "out", "dout", "dq", "dk", "dv"))
    b.stats, b.workspace, b.workspace_bytes = 0x10000, 0x10000, 1 << 60
    return (lib.dsqg_window_fwd(ctypes.byref(f), None), lib.dsqg_window_bwd_workspace_size(ctypes.byref(shape), ctypes.byref(n)),
            lib.dsqg_window_bwd(ctypes.byref(b), None))


@pytest.mark.parametrize("shape", [
    dict(B=1 << 14, H=1 << 10, Hkv=1, N=1), dict(B=1 << 10, H=1 << 10, Hkv=1, N=4096), dict(B=1 << 14, H=1 << 10, Hkv=1 << 10, N=1, D=128),
    dict(B=2 ** 31 - 1, H=2 ** 31 - 1, Hkv=1, N=1 << 30), dict(B=4096, H=4096, Hkv=4096, N=1, dtype=_lib.DSQG_F32),
])
def test_windows_past_the_grid(shape):
    assert _window(_shape(**shape)) == (_lib.DSQG_EUNSUPPORTED,) * 3


def test_window_backwards_past_the_grid():
    """Keys' and sinks' grids are larger than the forward's, which is not called here."""
    lib, n = _lib.load(), ctypes.c_size_t(0)

    def size(**kw):
        return lib.dsqg_window_bwd_workspace_size(ctypes.byref(_shape(**kw)), ctypes.byref(n))

    assert size(B=1 << 8, H=1 << 8, Hkv=1 << 8, N=4096, window=64, sinks=2048) == _lib.DSQG_EUNSUPPORTED
    assert size(B=1 << 8, H=1 << 8, Hkv=1 << 8, N=4096, window=64, sinks=0) == _lib.DSQG_OK
    assert size(B=1 << 8, H=1 << 8, Hkv=1 << 4, N=4096, window=64, sinks=2048) == _lib.DSQG_OK
    # What the header says always fits: B * H * ceil(N / 128) < 2^24 and B * Hkv * (N / 64 + 33) < 2^21.
    for dtype in (_lib.DSQG_F32, _lib.DSQG_BF16, _lib.DSQG_F16):
        for D in (32, 80, 128):
            for N in (1, 129, 5000, 1 << 20):
                most = min(((1 << 24) - 1) // -(-N // 128), ((1 << 21) - 1) // (N // 64 + 33))
                for sinks in (0, 1, 4, N // 2, N):
                    assert size(dtype=dtype, D=D, B=most, H=1, Hkv=1, N=N, window=1, sinks=sinks) == _lib.DSQG_OK


def test_what_rounding_took_off():
    """The 16-bit rest of the output: rows like any other's, and none for float32."""
    lib = _lib.load()
    f, b = _lib.WindowFwdArgs(), _lib.WindowBwdArgs()
    _fill(f, ("q", "k", "v", "out", "low"))
    _fill(b, ("q", "k", "v", "out", "dout", "low", "dq", "dk", "dv"))
    b.stats, b.workspace, b.workspace_bytes = 0x10000, 0x10000, 1 << 60
    for a, call in ((f, lib.dsqg_window_fwd), (b, lib.dsqg_window_bwd)):
        a.shape = _shape(dtype=_lib.DSQG_F32)
        assert call(ctypes.byref(a), None) == _lib.DSQG_EINVAL
        a.shape, a.low = _shape(), 0x10008
        assert call(ctypes.byref(a), None) == _lib.DSQG_EINVAL
        a.low, a.low_stride[2] = 0x10000, 32
        assert call(ctypes.byref(a), None) == _lib.DSQG_EINVAL


def test_trees_past_the_grid():
    lib, n = _lib.load(), ctypes.c_size_t(0)

    def call(**kw):
        a = _abi(**kw)
        return {lib.dsqg_paged_tree(ctypes.byref(a), None), lib.dsqg_paged_tree_workspace_size(ctypes.byref(a), ctypes.byref(n))}

    pool = dict(c_P=1, c_page=16)
    assert call(c_B=65535, c_Hkv=1024, H=1024, T=1, c_M=1, **pool) == {_lib.DSQG_EUNSUPPORTED}
    assert call(c_B=1, c_Hkv=1, H=1 << 16, T=64, **pool) == {_lib.DSQG_EUNSUPPORTED}        # 2^22 columns of one head
    a = _abi(c_B=1, c_Hkv=1, H=(1 << 21) - 32, T=1, **pool)
    assert lib.dsqg_paged_tree_workspace_size(ctypes.byref(a), ctypes.byref(n)) == _lib.DSQG_OK


def test_walks_past_the_grid():
    a = _lib.TreeAcceptArgs()
    a.B, a.T = 1 << 26, 1
    a.tokens = a.parents = a.picks = a.path = a.n = a.next = 0x10000
    assert _lib.load().dsqg_tree_accept(ctypes.byref(a), None) == _lib.DSQG_EUNSUPPORTED


@pytest.mark.parametrize("change", [
    dict(out=torch.zeros(2, 4, 8, 32).bfloat16()), dict(out=torch.zeros(2, 4, 9, 32)), dict(dout=torch.zeros(2, 2, 9, 32).bfloat16()),
    dict(stats=torch.zeros(2, 4, 9)), dict(stats=torch.zeros(2, 4, 9, 2).bfloat16()), dict(stats=torch.zeros(2, 4, 2, 9).transpose(2, 3)),
    dict(low=torch.zeros(2, 2, 9, 32).bfloat16()), dict(low=torch.zeros(2, 4, 9, 32)),
])
def test_window_backward_operands(change):
    """The backward's operator by itself: shapes and types are checked, and then only the GPU is missing."""
    def t(heads):
        return torch.zeros(2, heads, 9, 32).bfloat16()

    a = dict(q=t(4), k=t(2), v=t(2), lengths=None, out=t(4), stats=torch.zeros(2, 4, 9, 2), dout=t(4), window=4, sinks=1, softmax_scale=None,
             low=t(4))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.window_bwd(**a)
    with pytest.raises(AssertionError):
        ops.window_bwd(**{**a, **change})
