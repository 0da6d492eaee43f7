"""Attention within a window on the GPU, forward and gradients, against the 64-bit oracle within bounds that count the
kernels' roundings; layouts, ragged batches, infinities, captured and traced calls."""

import math

import pytest
import torch

from dwarf_amd import window_attention
from oracle import window_oracle as wo

pytestmark = pytest.mark.gpu
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF, F16]


def inputs(B, H, Hkv, N, D, dtype, seed=0, layout="tokens"):
    g = torch.Generator().manual_seed(seed)
    ch = torch.exp(0.5 * torch.randn(D, generator=g))

    def rows(heads, f=1.0):
        if layout == "tokens":  # head views of a projection's output
            return (torch.randn(B, N, heads, D, generator=g) * f).to(dtype).permute(0, 2, 1, 3)
        return (torch.randn(B, heads, N, D, generator=g) * f).to(dtype)

    return rows(H, 1.5), rows(Hkv, ch), rows(Hkv), rows(H)


def run(q, k, v, dout, window, sinks=0, lengths=None, scale=None, dev="cuda:0"):
    qd, kd, vd = (x.to(dev).requires_grad_() for x in (q, k, v))
    n = None if lengths is None else torch.as_tensor(lengths).to(dev)
    out = window_attention(qd, kd, vd, window, sinks, lengths=n, softmax_scale=scale)
    dq, dk, dv = torch.autograd.grad(out, (qd, kd, vd), dout.to(dev))
    with torch.no_grad():
        again = window_attention(qd, kd, vd, window, sinks, lengths=n, softmax_scale=scale)
        assert torch.allclose(out, again, rtol=0, atol=0, equal_nan=True)
    return dict(out=out.detach(), dq=dq, dk=dk, dv=dv)


def check(q, k, v, dout, window, sinks=0, lengths=None, scale=None):
    got = run(q, k, v, dout, window, sinks, lengths, scale)
    ref, tol = wo.forward_backward(q, k, v, dout, window, sinks, lengths, scale)
    for n, x in got.items():
        assert x.dtype == q.dtype and x.shape == ref[n].shape
        err = (x.double().cpu() - ref[n]).abs()
        bad = ~(err <= tol[n])
        assert not bad.any(), f"{n}: {int(bad.sum())} of {bad.numel()} beyond the bound, the first at " \
            f"{bad.nonzero()[0].tolist()}, worst {(err / tol[n].clamp(min=1e-300)).nan_to_num(1e9).max().item():.2f} of it"
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 80, 96, 128])
@pytest.mark.parametrize("N,window,sinks", [(150, 37, 3), (300, 64, 0), (65, 1000, 0)])
def test_types_and_head_dims(gpu_device, dtype, D, N, window, sinks):
    check(*inputs(2, 4, 2, N, D, dtype), window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 2, 15, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511])
def test_lengths(gpu_device, dtype, N):
    for window, sinks in ((1, 0), (1, 1), (7, 2), (33, 0), (N, 0), (max(1, N - 1), 5), (2 * N, 3)):
        check(*inputs(1, 2, 1, N, 32, dtype, seed=N), window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 100, 129, 300, 2 ** 40])
@pytest.mark.parametrize("sinks", [0, 1, 4, 32, 65, 130, 600, 2 ** 40])
def test_windows_and_sinks(gpu_device, dtype, window, sinks):
    check(*inputs(1, 2, 2, 420, 32, dtype, seed=window % 97), window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv", [(1, 1), (6, 2), (5, 1), (8, 1), (3, 3)])
def test_heads(gpu_device, dtype, H, Hkv):
    check(*inputs(2, H, Hkv, 190, 64, dtype), 50, 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ragged(gpu_device, dtype):
    """Rows behind the lengths, which may hold anything, are not seen; their outputs and gradients are zeros."""
    lengths = [200, 0, 1, 130, 64, -3, 1000, 199]
    q, k, v, dout = inputs(8, 4, 2, 200, 64, dtype)
    for junk in (None, math.nan, math.inf):
        if junk is not None:
            for x in (q, k, v, dout):
                for b, n in enumerate(lengths):
                    x[b, :, max(0, n):] = junk
        clean = [x.nan_to_num(0.0, 0.0, 0.0) for x in (q, k, v, dout)]
        for window, sinks in ((40, 3), (500, 0)):
            got = run(q, k, v, dout, window, sinks, lengths)
            ref, tol = wo.forward_backward(*clean, window, sinks, lengths)
            for n, x in got.items():
                assert ((x.double().cpu() - ref[n]).abs() <= tol[n]).all(), n
                for b, m in enumerate(lengths):
                    assert (x[b, :, max(0, m):] == 0).all(), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("D", [64, 80])
def test_infinities_stay_with_who_sees_them(gpu_device, dtype, value, D):
    N, at, window, sinks = 230, 100, 45, 2
    clean = inputs(1, 2, 1, N, D, dtype)
    want = run(*clean, window, sinks)
    seen = wo.sees(N, window, sinks)
    for which, name in enumerate(("q", "k", "v", "dout")):
        x = [t.clone() for t in clean]
        x[which][0, 0, at, 5] = value
        got = run(*x, window, sinks)
        # Queries that the row reaches, in the forward and, through them, in the backward.
        rows = torch.zeros(N, dtype=torch.bool)
        if name in ("q", "dout"):
            rows[at] = True
        else:
            rows = seen[:, at].clone()
        hit = {"out": rows if name != "dout" else torch.zeros_like(rows), "dq": rows}
        keys = (seen & rows[:, None]).any(0)
        hit["dk"] = hit["dv"] = keys
        for n, y in got.items():
            a, b = y[0].float().cpu(), want[n][0].float().cpu()
            free = ~hit[n]
            assert torch.isfinite(a[:, free]).all(), (name, n)
            most = 8 * torch.finfo(dtype).eps * b.abs().amax()
            assert ((a - b)[:, free].abs() <= most).all(), (name, n)
        if name == "v" and value == value:
            assert (got["out"][0, :, rows, 5] == value).all()
            assert torch.isfinite(got["out"][0, :, :, 6:]).all() and torch.isfinite(got["out"][0, :, :, :5]).all()
        if name == "dout" and value != value:
            assert torch.isnan(got["dv"][0, :, keys, 5]).all() and torch.isfinite(got["dv"][0, :, :, :5]).all()


@pytest.mark.parametrize("scale", [0.0, -0.4, 5.0, 1e-6])
def test_scales(gpu_device, scale):
    for dtype in DTYPES:
        check(*inputs(1, 2, 1, 170, 32, dtype), 60, 3, scale=scale)


def test_large_scores(gpu_device):
    """Scores past 2^24: the softmax picks the largest, and its gradients stay what they are."""
    for dtype in (F32, BF):
        q, k, v, dout = inputs(1, 1, 1, 100, 32, dtype)
        got = run(q * 2.0 ** 14, k * 2.0 ** 14, v, dout, 30, 1)
        s = (q[0, 0].double() @ k[0, 0].double().T).masked_fill(~wo.sees(100, 30, 1), -torch.inf)
        first, second = s.topk(2, -1).values.unbind(-1)
        sure = (first - second > 1e-2) | torch.isinf(second)  # (2^28 times that, far beyond the scores' rounding)
        out = got["out"][0, 0].cpu()
        assert sure.sum() > 80 and torch.equal(out[sure], v[0, 0][s.argmax(-1)][sure])
        assert all(torch.isfinite(x).all() for x in got.values())


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(gpu_device, dtype):
    want = run(*inputs(2, 4, 2, 140, 64, dtype, layout="plain"), 40, 3)
    q, k, v, dout = inputs(2, 4, 2, 140, 64, dtype, layout="plain")
    dev = "cuda:0"

    def odd(x):  # rows at odd places
        return torch.cat([torch.zeros_like(x[..., :1]), x], -1)[..., 1:]

    def wide(x):  # rows far apart
        y = torch.zeros(*x.shape[:3], 200, dtype=dtype, device=x.device)
        y[..., :64] = x
        return y[..., :64]

    for f in (odd, wide, lambda x: x.transpose(0, 3).contiguous().transpose(0, 3), lambda x: torch._neg_view(-x)):
        args = [f(x.to(dev)) for x in (q, k, v)]
        args = [x.detach().requires_grad_() for x in args]
        out = window_attention(*args, 40, 3)
        grads = torch.autograd.grad(out, args, f(dout.to(dev)))
        assert torch.equal(out, want["out"])
        for n, x in zip(("dq", "dk", "dv"), grads):
            assert torch.equal(x, want[n])


def test_expanded_inputs(gpu_device):
    """One key/value head for all, one prompt for all, one gradient for all: gradients are summed."""
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 4, 90, 32, generator=g)
    k, v = torch.randn(1, 1, 90, 32, generator=g), torch.randn(1, 1, 90, 32, generator=g)
    dev = "cuda:0"
    qd, kd, vd = (x.to(dev).requires_grad_() for x in (q, k, v))
    out = window_attention(qd, kd.expand(2, 4, 90, 32), vd.expand(2, 4, 90, 32), 20, 1)
    out.sum().backward()
    ref, tol = wo.forward_backward(q, k.expand(2, 4, 90, 32), v.expand(2, 4, 90, 32), torch.ones_like(q), 20, 1)
    assert ((qd.grad.double().cpu() - ref["dq"]).abs() <= tol["dq"]).all()
    for x, n in ((kd, "dk"), (vd, "dv")):
        want = ref[n].sum((0, 1))
        # Eight bounds and the roundings of torch's float32 sum of eight.
        assert ((x.grad[0, 0].double().cpu() - want).abs() <= tol[n].sum((0, 1)) + 8 * 2.0 ** -24 * ref[n].abs().sum((0, 1))).all()


def test_rows_without_a_stride(gpu_device):
    """Keys that are one row expanded along the positions."""
    g = torch.Generator().manual_seed(0)
    q, dout = torch.randn(1, 2, 70, 64, generator=g), torch.randn(1, 2, 70, 64, generator=g)
    row = torch.randn(1, 2, 1, 64, generator=g)
    check(q, row.expand(1, 2, 70, 64), row.expand(1, 2, 70, 64), dout, 20, 2)


@pytest.mark.parametrize("dtype,D,H,Hkv", [(BF, 128, 4, 1), (F32, 64, 2, 2), (F16, 80, 2, 1)])
def test_long(gpu_device, dtype, D, H, Hkv):
    for window, sinks in ((300, 4), (100, 260), (5000, 0)):
        check(*inputs(1, H, Hkv, 1500, D, dtype), window, sinks)


def test_repeats(gpu_device):
    args = inputs(2, 8, 2, 2000, 64, BF)
    a, b = run(*args, 200, 4), run(*args, 200, 4)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_against_differences(gpu_device):
    """The directional derivative of a weighted sum of float32 outputs, by central differences of the kernel itself."""
    g = torch.Generator().manual_seed(3)
    q, k, v, dout = inputs(1, 2, 1, 90, 32, F32, seed=3)
    got = run(q, k, v, dout, 25, 2)
    for which, name in ((0, "dq"), (1, "dk"), (2, "dv")):
        d = torch.randn((q, k, v)[which].shape, generator=g)
        h = 2.0 ** -6
        ends = []
        for s in (1, -1):
            x = [q, k, v]
            x[which] = x[which] + s * h * d
            out = window_attention(*[t.to("cuda:0") for t in x], 25, 2)
            ends.append((out.double().cpu() * dout.double()).sum())
        diff = (ends[0] - ends[1]) / (2 * h)
        want = (got[name].double().cpu() * d.double()).sum()
        # The exact function's own difference quotient says how far h is from the limit.
        exact = []
        for s in (1, -1):
            x = [q.double(), k.double(), v.double()]
            x[which] = x[which] + s * h * d.double()
            exact.append(sum((wo.attend(x[0][0, i], x[1][0, 0], x[2][0, 0], 25, 2) * dout[0, i].double()).sum() for i in range(2)))
        curve = ((exact[0] - exact[1]) / (2 * h) - want).abs()
        assert (diff - want).abs() <= curve + 1e-2 * want.abs().clamp(min=1.0)


def test_graph(gpu_device):
    """A captured forward and backward, replayed between eager ones."""
    dev = "cuda:0"
    for dtype in (BF, F32):
        args = [x.to(dev) for x in inputs(2, 4, 2, 700, 64, dtype)]
        lengths = torch.tensor([700, 333], device=dev)

        def step(q, k, v, dout):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            out = window_attention(*leaves, 100, 4, lengths=lengths)
            return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(*args)
        for seed in range(4):
            for x, y in zip(args, inputs(2, 4, 2, 700, 64, dtype, seed=seed)):
                x.copy_(y)
            lengths.copy_(torch.tensor([700 - 100 * seed, 333 + seed]))
            graph.replay()
            want = step(*args)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_other_stream(gpu_device):
    args = inputs(1, 2, 1, 300, 64, BF)
    want = run(*args, 50, 2)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run(*args, 50, 2)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_traced(gpu_device):
    q, k, v, dout = (x.to("cuda:0") for x in inputs(1, 4, 2, 120, 64, BF))
    f = torch.compile(lambda a, b, c: window_attention(a, b, c, 30, 2) * 2.0, backend="aot_eager")
    res = []
    for fn in (f, lambda a, b, c: window_attention(a, b, c, 30, 2) * 2.0):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = fn(*leaves)
        res.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_no_second_derivative(gpu_device):
    q = torch.randn(1, 1, 9, 32, device="cuda:0", requires_grad=True)
    out = window_attention(q, q, q, 4)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), q, create_graph=True)


def test_empty(gpu_device):
    for shape in ((0, 2, 5, 32), (2, 2, 0, 32), (2, 0, 5, 32)):
        q = torch.zeros(shape, device="cuda:0", requires_grad=True)
        out = window_attention(q, q, q, 4, 1)
        assert out.shape == shape
        assert torch.autograd.grad(out.sum(), q)[0].shape == shape
