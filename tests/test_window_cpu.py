"""Attention within a window without a GPU: the oracle against torch and its gradients, the refusals of the public
function, the C ABI's checks, traced shapes."""

import ctypes

import pytest
import torch

from dwarf_amd import _lib, window_attention
from oracle import window_oracle as wo


def test_oracle_is_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(20, 8, generator=g).double() for _ in range(3))
    ref = torch.nn.functional.scaled_dot_product_attention(q[None], k[None], v[None], is_causal=True)[0]
    assert torch.allclose(wo.attend(q, k, v, 20), ref, atol=1e-13, rtol=0)
    out = wo.attend(q, k, v, 3, 2)
    for i in range(20):
        rows = sorted(set(range(max(0, i - 2), i + 1)) | set(range(min(2, i + 1))))
        w = torch.softmax(q[i] @ k[rows].T * 8 ** -0.5, -1)
        assert torch.allclose(out[i], w @ v[rows], atol=1e-13, rtol=0)
    assert (wo.attend(q, k, v, 5, 0, 7)[7:] == 0).all()


def test_oracle_gradients():
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(s, 11, 6, generator=g) for s in (4, 2, 2, 4))
    ref, tol = wo.forward_backward(q[None], k[None], v[None], do[None], 4, 1, [9], 0.3)
    qd, kd, vd = (x.double().requires_grad_() for x in (q, k, v))
    out = torch.stack([wo.attend(qd[h], kd[h // 2], vd[h // 2], 4, 1, 9, 0.3) for h in range(4)])
    grads = torch.autograd.grad(out, (qd, kd, vd), do.double())
    assert torch.allclose(ref["out"][0], out, atol=1e-13)
    for n, x in zip(("dq", "dk", "dv"), grads):
        assert torch.allclose(ref[n][0], x, atol=1e-13) and (tol[n] >= 0).all()
    assert torch.autograd.gradcheck(lambda a, b, c: wo.attend(a, b, c, 3, 1), [x[0, :7].double().requires_grad_() for x in (q, k, v)])


def _t(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("args,kw", [
    ((_t(2, 4, 9, 32), _t(2, 3, 9, 32), _t(2, 3, 9, 32), 4), {}), ((_t(2, 4, 9, 32), _t(2, 2, 8, 32), _t(2, 2, 8, 32), 4), {}),
    ((_t(2, 4, 9, 32), _t(2, 2, 9, 32), _t(2, 4, 9, 32), 4), {}), ((_t(2, 4, 9, 32), _t(1, 2, 9, 32), _t(1, 2, 9, 32), 4), {}),
    ((_t(4, 9, 32), _t(4, 9, 32), _t(4, 9, 32), 4), {}), ((_t(2, 4, 9, 32), _t(2, 2, 9, 64), _t(2, 2, 9, 64), 4), {}),
    ((_t(2, 4, 9, 32), _t(2, 2, 9, 32, dtype=torch.float32), _t(2, 2, 9, 32), 4), {}),
    ((_t(2, 4, 9, 32, dtype=torch.float64),) * 3 + (4,), {}), ((_t(2, 4, 9, 32),) * 3 + (0,), {}), ((_t(2, 4, 9, 32),) * 3 + (-1,), {}),
    ((_t(2, 4, 9, 32),) * 3 + (4, -1), {}), ((_t(2, 4, 9, 32),) * 3 + (4,), dict(lengths=torch.zeros(3, dtype=torch.int64))),
    ((_t(2, 4, 9, 32),) * 3 + (4,), dict(lengths=torch.zeros(2))),
])
def test_refused(args, kw):
    with pytest.raises(AssertionError):
        window_attention(*args, **kw)


def test_only_the_gpu_is_missing():
    for grad in (False, True):
        q = torch.zeros(2, 4, 9, 32, requires_grad=grad)
        with pytest.raises(RuntimeError, match="GPU"):
            window_attention(q, q, q, 4, 1, lengths=torch.tensor([3, 9]))


def _shape(**kw):
    s = _lib.WindowShape()
    s.dtype, s.B, s.H, s.Hkv, s.N, s.D, s.window, s.softmax_scale = _lib.DSQG_BF16, 2, 4, 2, 50, 64, 8, 0.1
    for n, x in kw.items():
        setattr(s, n, x)
    return s


def _fill(a, names, **kw):
    for n in names:
        setattr(a, n, 0x10000)
        st = getattr(a, n + "_stride")
        st[0], st[1], st[2] = 4 * 50 * 64, 50 * 64, 64
    for n, x in kw.items():
        if n.endswith("_stride"):
            getattr(a, n)[2] = x
        else:
            setattr(a, n, x)


def test_abi_checks():
    lib = _lib.load()
    n = ctypes.c_size_t(0)

    def fwd(shape=None, **kw):
        a = _lib.WindowFwdArgs()
        a.shape = shape or _shape()
        _fill(a, ("q", "k", "v", "out"), **kw)
        return lib.dsqg_window_fwd(ctypes.byref(a), None)

    def bwd(shape=None, **kw):
        a = _lib.WindowBwdArgs()
        a.shape = shape or _shape()
        a.stats, a.workspace, a.workspace_bytes = 0x10000, 0x10000, 1 << 30
        _fill(a, ("q", "k", "v", "out", "dout", "dq", "dk", "dv"), **kw)
        return lib.dsqg_window_bwd(ctypes.byref(a), None)

    assert lib.dsqg_window_fwd(None, None) == lib.dsqg_window_bwd(None, None) == _lib.DSQG_EINVAL
    for call in (fwd, bwd):
        for bad in (dict(dtype=3), dict(B=-1), dict(H=3), dict(H=0), dict(Hkv=0), dict(N=-1), dict(D=0), dict(window=0), dict(sinks=-1)):
            assert call(_shape(**bad)) == _lib.DSQG_EINVAL, bad
        for bad in (dict(D=48), dict(N=(1 << 30) + 1), dict(B=1 << 20, H=1 << 10, Hkv=1 << 10)):
            assert call(_shape(**bad)) == _lib.DSQG_EUNSUPPORTED, bad
        assert call(_shape(N=0)) == _lib.DSQG_OK and call(_shape(B=0), q=None) == _lib.DSQG_OK
        for bad in (dict(q=None), dict(k=0x10008), dict(out=None), dict(v_stride=32), dict(q_stride=68), dict(k_stride=1 << 23),
                    dict(stats=0x10004)):
            assert call(**bad) == _lib.DSQG_EINVAL, bad
    for bad in (dict(dout=None), dict(dq=None), dict(dk=0x10002), dict(dv_stride=-64), dict(stats=None), dict(workspace=0x10010)):
        assert bwd(**bad) == _lib.DSQG_EINVAL, bad
    assert bwd(workspace=None) == bwd(workspace_bytes=100) == _lib.DSQG_EWORKSPACE
    assert lib.dsqg_window_bwd_workspace_size(None, ctypes.byref(n)) == _lib.DSQG_EINVAL
    assert lib.dsqg_window_bwd_workspace_size(ctypes.byref(_shape()), None) == _lib.DSQG_EINVAL
    size = {}
    for sinks in (0, 4, 300):
        assert lib.dsqg_window_bwd_workspace_size(ctypes.byref(_shape(N=20000, sinks=sinks)), ctypes.byref(n)) == _lib.DSQG_OK
        size[sinks] = n.value
    assert 0 < size[0] < size[4] <= 2 * size[300]
    assert lib.dsqg_window_bwd_workspace_size(ctypes.byref(_shape(N=0)), ctypes.byref(n)) == _lib.DSQG_OK and n.value == 0


def test_traced_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from dwarf_amd import ops
    with FakeTensorMode():
        q, k = torch.empty(2, 6, 9, 32, device="cuda"), torch.empty(2, 2, 9, 32, device="cuda")
        out = window_attention(q, k, k, 4, 1)
        assert out.shape == (2, 6, 9, 32) and out.stride() == (9 * 6 * 32, 32, 6 * 32, 1)
        stats = torch.empty(2, 6, 9, 2, device="cuda")
        dq, dk, dv = ops.window_bwd(q, k, k, None, out, stats, q, 4, 1, None)
        assert dq.shape == q.shape and dk.shape == dv.shape == k.shape and dk.stride() == (9 * 2 * 32, 32, 2 * 32, 1)


def test_structs_match_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    header = Path(__file__).resolve().parents[1] / "include" / "dsqg.h"
    probes = {"dsqg_window_shape": _lib.WindowShape, "dsqg_window_fwd_args": _lib.WindowFwdArgs, "dsqg_window_bwd_args": _lib.WindowBwdArgs}
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
