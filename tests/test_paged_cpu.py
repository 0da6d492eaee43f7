"""The paged key/value cache without a GPU: the oracle against torch's own conversions and attention, the
refusals of the public functions, and the C ABI's argument checks."""

import ctypes
import math

import pytest
import torch

import dwarf_amd
from dwarf_amd import PagedKVCache, _lib
from oracle import paged_oracle as po

BF, I8, E4 = torch.bfloat16, torch.int8, torch.float8_e4m3fn


# ---- The oracle. -----------------------------------------------------------------------------------

@pytest.mark.parametrize("kv", [E4, I8])
def test_oracle_encoding(kv):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(300, 32, generator=g) * torch.exp(3 * torch.randn(300, 1, generator=g))
    codes, e = po.encode(x, kv)
    top, scale = po.LARGEST[kv], 2.0 ** (e.double() - 127)
    size = x.abs().amax(-1).double()
    assert (size <= top * scale).all() and (size > top * scale / 2).all()
    y = x.double() / scale[:, None]
    if kv == E4:
        assert torch.equal(codes, y.float().to(E4).double())
        small = torch.arange(-128, 128).to(torch.int8).view(E4).double()  # every code stands for itself
        assert torch.isin(codes, small).all()
    else:
        assert torch.equal(codes, y.round())
    # Nothing is nearer than half a step.
    step = 1.0 if kv == I8 else torch.maximum(y.abs() * 2.0 ** -3, torch.tensor(2.0 ** -9, dtype=torch.float64))
    assert ((codes - y).abs() <= step / 2).all()


def test_oracle_encoding_at_the_edges():
    for kv, top in po.LARGEST.items():
        assert po.encode_row([0.0, -0.0], kv) == ([0.0, 0.0], 0)
        assert po.encode_row([top, -1.0], kv) == ([top, -1.0], 127)
        assert po.encode_row([math.nextafter(top, math.inf), 0.0], kv)[1] == 128
        assert po.encode_row([math.inf, 1.0], kv)[1] == po.encode_row([1.0, math.nan], kv)[1] == 255
        assert po.encode_row([2.0 ** -149, 0.0], kv)[1] == 0
    assert po.encode_row([127.0, 2.5, 3.5, -0.5], I8)[0] == [127, 2, 4, 0]


def test_oracle_attention():
    g = torch.Generator().manual_seed(2)
    q, k, v = torch.randn(6, 8, generator=g), torch.randn(2, 11, 8, generator=g), torch.randn(2, 11, 8, generator=g)
    out, mass, size = po.attend(q, k.double(), v.double(), 8 ** -0.5)
    ref = torch.nn.functional.scaled_dot_product_attention(
        q[None, :, None].double(), k.repeat_interleave(3, 0)[None].double(), v.repeat_interleave(3, 0)[None].double())
    assert torch.allclose(out, ref[0, :, 0], rtol=0, atol=1e-13)
    assert (mass[:, 0] >= out.abs()).all() and (mass[:, 1] >= mass[:, 0]).all() and size.shape == (6, 1)


def test_oracle_sequence():
    pages = torch.arange(4 * 1 * 16 * 2, dtype=torch.float32).view(4, 1, 16, 2)
    table = torch.tensor([[2, 0, -1], [1, 4, 3]], dtype=torch.int32)
    x = po.sequence(pages, table, 0, 20)
    assert torch.equal(x[0, :16], pages[2, 0].double()) and torch.equal(x[0, 16:], pages[0, 0, :4].double())
    assert torch.isnan(po.sequence(pages, table, 0, 33)[0, 32]).all()
    x = po.sequence(pages, table, 1, 50)
    assert torch.isnan(x[0, 16:32]).all() and torch.isnan(x[0, 48:]).all() and torch.equal(x[0, 32:48], pages[3, 0].double())


# ---- Refusals of the public functions. ---------------------------------------------------------------

def _pool(P=4, H=2, page=16, D=32, dtype=BF):
    x = torch.zeros(P, H, page, D, dtype=dtype)
    if x.element_size() > 1:
        return x, x.clone(), None, None
    s = torch.zeros(P, H, page, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return x, x.clone(), s, s.clone()


def _calls(B=2, H=2, G=1, D=32, N=3, dtype=BF, kv=BF, **pool):
    """The three calls with arguments that only lack a GPU, as (function, arguments) by name."""
    kp, vp, ks, vs = _pool(H=H, D=D, dtype=kv, **pool)
    table, pos = torch.zeros(B, 2, dtype=torch.int32), torch.zeros(B, dtype=torch.int64)
    s = dict(k_pages=kp, v_pages=vp, page_table=table, k_scale=ks, v_scale=vs)
    row = lambda *shape: torch.zeros(*shape, dtype=dtype)
    return {
        "write": (dwarf_amd.paged_kv_write, dict(k=row(B, H, N, D), v=row(B, H, N, D), pos=pos, **s)),
        "step": (dwarf_amd.paged_decode_step, dict(q=row(B, H * G, D), k_new=row(B, H, D), v_new=row(B, H, D), pos=pos, **s)),
        "read": (dwarf_amd.paged_kv_read, dict(lengths=pos, max_len=20, **s)),
    }


@pytest.mark.parametrize("name", ["write", "step", "read"])
@pytest.mark.parametrize("kv", [BF, E4, I8])
def test_refuses_cpu_tensors(name, kv):
    fn, args = _calls(kv=kv)[name]
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fn(**args)


z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)
E8 = lambda *s: torch.zeros(*s, dtype=torch.uint8).view(torch.float8_e8m0fnu)
BAD = [
    ("any", dict(v_pages=z(4, 2, 16, 64)), "same shape"),
    ("any", dict(v_pages=z(4, 2, 16, 32, dtype=torch.float32)), "same shape and dtype"),
    ("any", dict(k_pages=z(4, 2, 16)), r"\[P,H,page,D\]"),
    ("any", dict(k_pages=z(4, 2, 24, 32), v_pages=z(4, 2, 24, 32)), "power of two"),
    ("any", dict(k_pages=z(4, 2, 8, 32), v_pages=z(4, 2, 8, 32)), "power of two"),
    ("any", dict(k_pages=z(4, 2, 16, 32, dtype=torch.float64), v_pages=z(4, 2, 16, 32, dtype=torch.float64)), "pages must be"),
    ("any", dict(k_scale=E8(4, 2, 16), v_scale=E8(4, 2, 16)), "8-bit pages"),
    ("any", dict(page_table=z(2, 2, dtype=torch.int64)), "int32"),
    ("any", dict(page_table=z(4, dtype=torch.int32)), "int32"),
    ("write", dict(v=z(2, 2, 4, 32)), "same shape"),
    ("write", dict(v=z(2, 2, 3, 32, dtype=torch.float16)), "share a dtype"),
    ("write", dict(k=z(2, 2, 3, 32, dtype=torch.float32), v=z(2, 2, 3, 32, dtype=torch.float32)), "do not go into"),
    ("write", dict(k=z(2, 2, 3, 32, dtype=torch.float64), v=z(2, 2, 3, 32, dtype=torch.float64)), "rows must be"),
    ("write", dict(k=z(1, 2, 3, 32), v=z(1, 2, 3, 32)), "k and v must be"),
    ("write", dict(k=z(2, 1, 3, 32), v=z(2, 1, 3, 32)), "k and v must be"),
    ("step", dict(q=z(2, 3, 32)), "multiple of 2"),
    ("step", dict(q=z(2, 0, 32)), "multiple of 2"),
    ("step", dict(q=z(2, 2, 64)), "q must be"),
    ("step", dict(q=z(1, 2, 32)), "q must be"),
    ("step", dict(q=z(2, 2, 32, dtype=torch.float16)), "do not go with"),
    ("step", dict(k_new=None), "go together"),
    ("step", dict(k_new=z(2, 4, 32)), "k_new and v_new must be"),
    ("step", dict(v_new=z(2, 2, 32, dtype=torch.float32)), "k_new and v_new must be"),
]


@pytest.mark.parametrize("name,bad,match", [(n, b, m) for n, b, m in BAD for n in (["write", "step", "read"] if n == "any" else [n])])
def test_refuses_bad_arguments(name, bad, match):
    fn, args = _calls()[name]
    # (Arguments are refused before the device is looked at, or the device is what is refused.)
    with pytest.raises((AssertionError, RuntimeError), match=match + "|ROCm GPU") as e:
        fn(**{**args, **bad})
    if not match.startswith(("do not", "multiple", "q must", "k_new", "k and v must")):
        assert e.type is AssertionError


@pytest.mark.parametrize("name", ["write", "step", "read"])
def test_8_bit_pages_need_their_scales(name):
    for bad in (dict(k_scale=None), dict(v_scale=None), dict(k_scale=E8(4, 2, 8), v_scale=E8(4, 2, 8)),
                dict(k_scale=z(4, 2, 16, dtype=torch.float32), v_scale=z(4, 2, 16, dtype=torch.float32))):
        fn, args = _calls(kv=I8)[name]
        with pytest.raises(AssertionError, match="scale"):
            fn(**{**args, **bad})


def test_refuses_gradients():
    for name, key in (("write", "k"), ("write", "v"), ("step", "q"), ("step", "v_new"), ("step", "k_pages"), ("read", "v_pages")):
        fn, args = _calls()[name]
        with pytest.raises(RuntimeError, match="no gradient"):
            fn(**{**args, key: args[key].requires_grad_(True)})


def test_cache_class_on_the_host():
    c = PagedKVCache(3, 2, 32, 100, device="cpu", page_size=16)
    assert c.k_pages.shape == (21, 2, 16, 32) and c.k_scale is None and c.page_table.tolist()[2] == list(range(14, 21))
    c = PagedKVCache(1, 2, 80, 64, dtype=torch.float16, device="cpu", kv_dtype=I8)
    assert c.v_pages.dtype == I8 and c.v_scale.dtype == torch.float8_e8m0fnu and c.v_scale.shape == (1, 2, 64)
    for bad in (dict(max_len=0), dict(D=48), dict(kv_dtype=torch.float32), dict(kv_dtype=torch.uint8)):
        with pytest.raises(AssertionError):
            PagedKVCache(**{**dict(B=1, H=1, D=32, max_len=10, device="cpu"), **bad})
    with pytest.raises(AssertionError, match="exceeds the cache"):
        c.prefill(torch.zeros(1, 2, 65, 80), torch.zeros(1, 2, 65, 80))


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        fn, args = _calls(G=3)["step"]
        assert fn(**args).shape == (2, 6, 32)
        fn, args = _calls(kv=E4)["read"]
        k, v = fn(**args)
        assert k.shape == v.shape == (2, 2, 20, 32) and k.dtype == BF
        fn, args = _calls(kv=I8)["write"]
        assert fn(**args) is None


# ---- The C ABI. ------------------------------------------------------------------------------------------

def _cache_args(kv=None):
    c = _lib.PagedCache()
    c.dtype = _lib.DSQG_BF16
    c.cache_dtype = c.dtype if kv is None else kv
    c.B, c.Hkv, c.D, c.P, c.page, c.M = 2, 3, 64, 7, 32, 4
    c.k_pages = c.v_pages = 0x10000
    c.k_stride = c.v_stride = (3 * 32 * 64, 32 * 64, 64)
    if kv is not None:
        c.k_scale = c.v_scale = 0x20001
        c.k_scale_stride = c.v_scale_stride = (96, 32, 1)
    c.page_table, c.table_stride = 0x30000, 4
    return c


def _abi(kv=None):
    """(entry point's name, valid arguments) of the three calls; never launched as they are."""
    w = _lib.PagedWriteArgs(cache=_cache_args(kv), N=5, k=0x1000, k_stride=(960, 320, 64), v=0x1000,
                            v_stride=(960, 320, 64), pos=0x100, counts=None)
    r = _lib.PagedReadArgs(cache=_cache_args(kv), T=9, lengths=0x100, k=0x1000, v=0x1000)
    d = _lib.PagedDecodeArgs(cache=_cache_args(kv), H=6, softmax_scale=0.1, q=0x1000, q_stride=(384, 64), k_new=0x1000,
                             k_new_stride=(192, 64), v_new=0x1000, v_new_stride=(192, 64), pos=0x100, out=0x1000)
    return {"dsqg_paged_write": w, "dsqg_paged_read": r, "dsqg_paged_decode": d}


def _call(name, a):
    return getattr(_lib.load(), name)(ctypes.byref(a), None)


NAMES = ["dsqg_paged_write", "dsqg_paged_read", "dsqg_paged_decode"]


@pytest.mark.parametrize("name", NAMES)
def test_abi_checks_the_cache(name):
    for field, value, want in (
            ("dtype", 3, 1), ("dtype", -1, 1), ("cache_dtype", 5, 1), ("B", -1, 1), ("Hkv", -1, 1), ("D", 0, 1), ("P", -1, 1),
            ("M", -1, 1), ("page", 24, 1), ("page", 0, 1), ("page", 8, 2), ("page", 1 << 17, 2), ("D", 48, 2), ("M", 1 << 26, 2),
            ("B", 70000, 2), ("Hkv", 70000, 2), ("P", 0, 1), ("k_pages", None, 1), ("v_pages", 0x10008, 1),
            ("k_stride", (3 * 32 * 64, 32 * 64, 68), 1), ("v_stride", (-64, 32 * 64, 64), 1),
            ("k_stride", (0, 32 * 64, 64), 1), ("v_stride", (3 * 32 * 64, 32 * 64, 32), 1),
            ("k_stride", (2 * 32 * 64, 32 * 64, 64), 1), ("page_table", None, 1), ("table_stride", -1, 1)):
        a = _abi()[name]
        c = _lib.PagedCache.from_buffer_copy(a.cache)
        setattr(c, field, value)
        a.cache = c
        if name == "dsqg_paged_decode":
            a.H = 2 * max(c.Hkv, 0)
        assert _call(name, a) == want, (field, value)
    for field, value in (("k_scale", None), ("v_scale", None), ("v_scale_stride", (96, 16, 1)), ("k_scale_stride", (96, 32, -1))):
        a = _abi(_lib.DSQG_INT8)[name]
        c = _lib.PagedCache.from_buffer_copy(a.cache)
        setattr(c, field, value)
        a.cache = c
        assert _call(name, a) == _lib.DSQG_EINVAL, field
    assert getattr(_lib.load(), name)(None, None) == _lib.DSQG_EINVAL
    a = _abi()[name]
    c = _lib.PagedCache.from_buffer_copy(a.cache)
    c.B, c.k_pages = 0, None
    a.cache = c
    assert _call(name, a) == _lib.DSQG_OK  # nothing to do, nothing to check


@pytest.mark.parametrize("name,bad", [
    ("dsqg_paged_write", dict(N=-1)), ("dsqg_paged_write", dict(k=None)), ("dsqg_paged_write", dict(v=0x1008)),
    ("dsqg_paged_write", dict(pos=None)), ("dsqg_paged_write", dict(k_stride=(960, 320, 68))),
    ("dsqg_paged_write", dict(v_stride=(960, -320, 64))), ("dsqg_paged_read", dict(T=-1)),
    ("dsqg_paged_read", dict(lengths=None)), ("dsqg_paged_read", dict(k=0x1004)), ("dsqg_paged_read", dict(v=None)),
    ("dsqg_paged_decode", dict(H=5)), ("dsqg_paged_decode", dict(H=-3)), ("dsqg_paged_decode", dict(H=0)), ("dsqg_paged_decode", dict(q=None)),
    ("dsqg_paged_decode", dict(q_stride=(384, 60))), ("dsqg_paged_decode", dict(k_new=None)),
    ("dsqg_paged_decode", dict(v_new=0x1004)), ("dsqg_paged_decode", dict(pos=None)), ("dsqg_paged_decode", dict(out=0x1002)),
])
def test_abi_checks_the_call(name, bad):
    a = _abi()[name]
    for k, v in bad.items():
        setattr(a, k, v)
    assert _call(name, a) == _lib.DSQG_EINVAL


@pytest.mark.parametrize("name", ["dsqg_paged_write", "dsqg_paged_decode"])
def test_abi_refuses_pages_of_another_type(name):
    a = _abi()[name]
    c = _lib.PagedCache.from_buffer_copy(a.cache)
    c.cache_dtype = _lib.DSQG_F16
    a.cache = c
    assert _call(name, a) == _lib.DSQG_EINVAL


def test_abi_workspace():
    lib, n = _lib.load(), ctypes.c_size_t(1)
    a = _abi()["dsqg_paged_decode"]
    assert lib.dsqg_paged_decode_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 0
    assert lib.dsqg_paged_decode_workspace_size(ctypes.byref(a), None) == _lib.DSQG_EINVAL
    c = _lib.PagedCache.from_buffer_copy(a.cache)
    c.B, c.M = 1, 4096
    a.cache = c
    assert lib.dsqg_paged_decode_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value > 0
    assert _call("dsqg_paged_decode", a) == _lib.DSQG_EWORKSPACE
    a.workspace, a.workspace_bytes = 0x10000, n.value - 1
    assert _call("dsqg_paged_decode", a) == _lib.DSQG_EWORKSPACE
    a.workspace, a.workspace_bytes = 0x10080, n.value
    assert _call("dsqg_paged_decode", a) == _lib.DSQG_EINVAL


def test_ctypes_layout_matches_c(tmp_path):
    import subprocess
    from pathlib import Path
    header = Path(__file__).resolve().parents[1] / "include" / "dsqg.h"
    probes = {"dsqg_paged_cache": _lib.PagedCache, "dsqg_paged_write_args": _lib.PagedWriteArgs,
              "dsqg_paged_read_args": _lib.PagedReadArgs, "dsqg_paged_decode_args": _lib.PagedDecodeArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    for c, s in probes.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in s._fields_]
    src, exe = tmp_path / "p.c", tmp_path / "p"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    want = []
    for s in probes.values():
        want += [ctypes.sizeof(s)] + [getattr(s, f).offset for f, _ in s._fields_]
    assert got == want


# ---- Refusals by their own message, whatever the device. ------------------------------------------------------------

@pytest.mark.parametrize("name,bad,match", [(n, b, m) for n, b, m in BAD for n in (["write", "step", "read"] if n == "any" else [n])])
def test_refuses_bad_arguments_by_name(name, bad, match):
    """Shapes and types are looked at before the device, so each check is the one that refuses."""
    fn, args = _calls()[name]
    with pytest.raises(AssertionError, match=match):
        fn(**{**args, **bad})


@pytest.mark.parametrize("bad,match", [
    (dict(k=z(2, 2, 3, 64), v=z(2, 2, 3, 64)), "k and v must be"), (dict(k=z(2, 4, 3, 32), v=z(2, 4, 3, 32)), "k and v must be"),
    (dict(k=z(3, 2, 3, 32), v=z(3, 2, 3, 32)), "k and v must be"), (dict(k=z(2, 2, 32), v=z(2, 2, 32)), "same shape")])
def test_write_refuses_rows_of_another_cache(bad, match):
    fn, args = _calls()["write"]
    with pytest.raises(AssertionError, match=match):
        fn(**{**args, **bad})


@pytest.mark.parametrize("bad,match", [
    (dict(q=z(3, 2, 32)), "q must be"), (dict(q=z(2, 2)), "q must be"), (dict(k_new=z(2, 1, 32), v_new=z(2, 1, 32)), "k_new and v_new"),
    (dict(k_new=z(1, 2, 32)), "k_new and v_new"), (dict(v_new=z(2, 2, 64)), "k_new and v_new"), (dict(v_new=None), "go together")])
def test_step_refuses_rows_of_another_cache(bad, match):
    fn, args = _calls()["step"]
    with pytest.raises(AssertionError, match=match):
        fn(**{**args, **bad})


# ---- Counts of narrow types. -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("name", ["prefill", "write"])
def test_cache_takes_counts_of_any_integer_type(name, dtype):
    """A prompt of more rows than the counts' type can say (the call goes on until it finds no GPU)."""
    c = PagedKVCache(2, 1, 32, 70000, device="cpu")
    rows = torch.zeros(2, 1, 1, 32, dtype=BF).expand(2, 1, 70000, 32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        getattr(c, name)(rows, rows, torch.tensor([100, 7], dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bool])
@pytest.mark.parametrize("name", ["prefill", "write"])
def test_cache_refuses_counts_that_are_no_integers(name, dtype):
    c = PagedKVCache(2, 1, 32, 100, device="cpu")
    rows = torch.zeros(2, 1, 5, 32, dtype=BF)
    with pytest.raises(AssertionError, match="counts must be"):
        getattr(c, name)(rows, rows, torch.ones(2, dtype=dtype))


# ---- Calls of very many rows. ----------------------------------------------------------------------------------------

def test_refuses_more_rows_than_memory_has():
    fn, args = _calls()["read"]
    for bad in (-1, 2 ** 30, 2 ** 31, 2 ** 62):
        with pytest.raises(AssertionError, match="max_len must be"):
            fn(**{**args, "max_len": bad})
    fn, args = _calls()["write"]
    rows = z(1, 1, 1, 32).expand(2, 2, 2 ** 30, 32)
    with pytest.raises(AssertionError, match="less than 2\\^31 rows"):
        fn(**{**args, "k": rows, "v": rows})
    for name, field in (("dsqg_paged_write", "N"), ("dsqg_paged_read", "T")):
        a = _abi()[name]
        setattr(a, field, 2 ** 31 // 3 + 1)
        assert _call(name, a) == _lib.DSQG_EUNSUPPORTED


# ---- How a step is split. --------------------------------------------------------------------------------------------

CODE = {torch.float32: 0, BF: 1, torch.float16: 2, E4: 3, I8: 4}


def split_of(dtype, kv, B, Hkv, H, D, page, M):
    """("one", 0), ("chunks", their number) or ("shares", their number): a step's split, from the size of its
    workspace (each part has D + 2 floats a head, each unit two integers)."""
    c = _lib.PagedCache()
    c.dtype, c.cache_dtype, c.B, c.Hkv, c.D, c.P, c.page, c.M = CODE[dtype], CODE[kv or dtype], B, Hkv, D, 64, page, M
    c.k_pages = c.v_pages = 0x10000
    c.k_stride = c.v_stride = (Hkv * page * D, page * D, D)
    if kv is not None:
        c.k_scale = c.v_scale = 0x20000
        c.k_scale_stride = c.v_scale_stride = (Hkv * page, page, 1)
    c.page_table, c.table_stride = 0x30000, M
    a, n = _lib.PagedDecodeArgs(cache=c, H=H), ctypes.c_size_t(0)
    assert _lib.load().dsqg_paged_decode_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 0
    if n.value == 0:
        return "one", 0
    G = H // Hkv
    heads = min(G, 16) if dtype != torch.float32 else 1 if G == 1 else 2 if G == 2 or D in (80, 96) else 4
    units = B * Hkv * -(-G // heads)
    parts, rest = divmod(n.value - units * 8, heads * (D + 2) * 4)
    assert rest == 0
    places = 256 * (4 if D <= 64 else 3)
    if parts == places + units:
        return "shares", places
    assert parts % units == 0
    return "chunks", parts // units


@pytest.mark.parametrize("want,B,Hkv,G,D,dtype,kv,page,M", [
    ("one", 1, 8, 1, 32, BF, None, 64, 2), ("one", 512, 1, 1, 64, BF, None, 64, 64), ("chunks", 1, 8, 1, 64, BF, None, 64, 2048),
    ("chunks", 4, 8, 1, 32, torch.float32, None, 64, 32), ("chunks", 5, 3, 5, 80, torch.float16, I8, 64, 80),
    ("shares", 64, 8, 4, 128, BF, E4, 128, 64), ("shares", 64, 8, 4, 128, torch.float16, I8, 128, 64),
    ("shares", 64, 8, 1, 64, BF, None, 64, 125), ("chunks", 64, 8, 4, 128, BF, None, 128, 64),
    ("chunks", 64, 8, 1, 64, torch.float32, None, 64, 125)])
def test_split(want, B, Hkv, G, D, dtype, kv, page, M):
    """One workgroup a unit under short tables, chunks under long ones, equal shares of large batches, but not of
    16-bit rows of 128 and not of float32."""
    assert split_of(dtype, kv, B, Hkv, Hkv * G, D, page, M)[0] == want
