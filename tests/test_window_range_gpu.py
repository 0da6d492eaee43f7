"""Attention within a window on the GPU at the ends of its range: huge scores, the largest values, few keys, float16's
small and large gradients, and batches whose workgroups have eight waves."""

import pytest
import torch

from dwarf_amd import window_attention
from oracle import window_oracle as wo
from tests.test_window_gpu import BF, F16, F32, check, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF, F32])
@pytest.mark.parametrize("power", [14, 18, 20, 21, 22, 23, 24, 25, 26, 27, 28, 30])
def test_huge_scores(gpu_device, dtype, power):
    """Scores up to 2^36, whose steps are larger than what their weights are moved by: the largest one's row comes out as it
    is.  Sums of |q||k| are below 2^8, so that a score is off by 40 2^-24 2^8 times the scale at most, and one that is ahead by 2^8
    besides leaves the others exp(-2^8) of its weight: nothing."""
    q, k, v, dout = inputs(1, 1, 1, 300, 32, dtype)
    size = (q[0, 0].double().abs() @ k[0, 0].double().abs().T).max()
    assert size < 2 ** 8
    got = run(q, k, v, dout, 40, 2, scale=2.0 ** power)
    s = (q[0, 0].double() @ k[0, 0].double().T).masked_fill(~wo.sees(300, 40, 2), -torch.inf)
    first, second = s.topk(2, -1).values.unbind(-1)
    sure = first - second > 2 * 40 * 2.0 ** -16 + 2.0 ** (8 - power)
    out = got["out"][0, 0].cpu()
    assert sure.sum() > 200 and torch.equal(out[sure], v[0, 0][s.argmax(-1)][sure])
    assert all(torch.isfinite(x).all() for x in got.values())


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("D", [32, 80, 128])
@pytest.mark.parametrize("flat", [True, False])
def test_largest_values(gpu_device, dtype, D, flat):
    """Values of half the type's largest to 0.95 of it, of one sign in each element: their means are as large, and finite."""
    q, k, v, dout = inputs(2, 2, 1, 300, D, dtype)
    sign = torch.where(torch.arange(D) % 3 == 0, -1.0, 1.0)
    v = (sign * (1.0 + 0.9 * torch.rand(2, 1, 300, D, generator=torch.Generator().manual_seed(D)))).to(dtype)
    v = v * 2.0 ** (15 if dtype == F16 else 127)
    # (Gradients pass by products of dout with those, which are to be numbers too.)
    got = check(q * (0.0 if flat else 1.0), k, v, dout * 2.0 ** (-10 if dtype == F16 else -20), 200, 3, lengths=[300, 77])
    assert all(torch.isfinite(x).all() for x in got.values())
    assert got["out"][0].float().abs().amin() >= (2.0 ** 15 if dtype == F16 else 2.0 ** 127) * (1 - 2.0 ** -7)


def far_off(got, ref):
    """|got - ref| over |ref|, 2-norms."""
    return ((got.double().cpu() - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [32, 80, 128])
@pytest.mark.parametrize("window,sinks", [(1, 1), (2, 0), (3, 0), (8, 1)])
def test_gradients_of_few_keys(gpu_device, dtype, D, window, sinks):
    """Three roundings make dq and dk, of at most half a step e each: the result's, dS's, and the weights' behind dout . out.
    Even ones from -e to e are e / sqrt(3) in the mean, and three of them e.  (Were dout . out taken from the rounded output, its
    error of e |dout||out| / sqrt(D) would be larger than the dS of queries with nearly all their weight on one key.)"""
    q, k, v, dout = inputs(1, 2, 1, 600, D, dtype)
    got = run(q, k, v, dout, window, sinks)
    ref, _ = wo.forward_backward(q, k, v, dout, window, sinks)
    for n in ("dq", "dk", "dv"):
        assert far_off(got[n], ref[n]) <= torch.finfo(dtype).eps / 2, n


@pytest.mark.parametrize("size", [1e-4, 1.0, 1e3])
@pytest.mark.parametrize("D,G", [(32, 1), (64, 2), (80, 1), (128, 2)])
@pytest.mark.parametrize("sinks", [0, 4])
def test_float16_gradients_of_any_size(gpu_device, size, D, G, sinks):
    """A long window's weights and small gradients lie far below float16's normal numbers: both are brought up before they are
    rounded, so that the errors are those of ``test_gradients_of_few_keys``, and for dv those of two roundings."""
    q, k, v, dout = inputs(1, G, 1, 1500, D, F16)
    dout = (dout.float() * size).half()
    got = run(q, k, v, dout, 1024, sinks)
    ref, _ = wo.forward_backward(q, k, v, dout, 1024, sinks)
    # (Results below 2^-14 are off by half their smallest step, 2^-25, each.)
    for n in ("dq", "dk", "dv"):
        assert far_off(got[n], ref[n]) <= torch.finfo(F16).eps / 2 + 2.0 ** -25 * ref[n].numel() ** 0.5 / ref[n].norm(), n


@pytest.mark.parametrize("D", [32, 80, 128])
def test_float16_gradients_past_the_largest_on_the_way(gpu_device, D):
    """Score gradients above 65504 in front of small keys and queries: the results fit."""
    q, k, v, dout = inputs(1, 2, 1, 400, D, F16)
    q, k, v, dout = (x.float() * f for x, f in ((q, 2.0 ** -6), (k, 2.0 ** -6), (v, 16.0), (dout, 2e3)))
    dout[:, :, 200:] *= 2.0 ** -12  # and others that are small, before and behind them
    dout[:, :, :100] *= 2.0 ** -20
    q, k, v, dout = (x.half() for x in (q, k, v, dout))
    ref, _ = wo.forward_backward(q, k, v, dout, 3, 1)
    # (Weights of three keys are a third each, more or less: a score's gradient, that of dout . v's distance from their mean.)
    dp = torch.stack([(dout[0, 0, i].double() * v[0, 0, i - 2:i + 1].double()).sum(-1) for i in range(100, 200)])
    assert ((dp - dp.mean(1, keepdim=True)).abs() / 3 > 65504).sum() > 20
    assert all(x.abs().max() < 65504 for x in ref.values())
    got = run(q, k, v, dout, 3, 1)
    for n in ("dq", "dk", "dv"):
        assert far_off(got[n], ref[n]) <= torch.finfo(F16).eps / 2, n
        for rows in (slice(2, 90), slice(220, 400)):  # rows of small gradients on their own
            a, b = got[n][:, :, rows], ref[n][:, :, rows]
            assert far_off(a, b) <= torch.finfo(F16).eps / 2 + 2.0 ** -25 * b.numel() ** 0.5 / b.norm(), (n, rows)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [80, 96, 128])
@pytest.mark.parametrize("window,sinks", [(40, 3), (7, 0), (300, 0)])
def test_many_short_heads(gpu_device, dtype, D, window, sinks):
    """Rows above 64 elements of 16 bits in 512 and more blocks of 256 queries: workgroups of eight waves, in the forward and for dq."""
    B, H, N = 32, 16, 130
    assert B * H * -(-N // 256) >= 512
    lengths = [N - 4 * b if b % 3 else N for b in range(B)]
    check(*inputs(B, H, 4, N, D, dtype), window, sinks, lengths)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (F16, 80)])
def test_long_rows_of_eight_waves(gpu_device, dtype, D):
    """... whose queries are several blocks, with tiles in front of the window and sinks beyond it; a few heads of them."""
    B, H, N, window, sinks = 8, 16, 1100, 150, 70
    assert B * H * -(-N // 256) >= 512
    q, k, v, dout = inputs(B, H, 4, N, D, dtype)
    got = run(q, k, v, dout, window, sinks)
    for b, hk in ((0, 0), (5, 3)):
        ref, tol = wo.forward_backward(q[b:b + 1, 4 * hk:4 * hk + 4], k[b:b + 1, hk:hk + 1], v[b:b + 1, hk:hk + 1],
                                       dout[b:b + 1, 4 * hk:4 * hk + 4], window, sinks)
        for n, x in got.items():
            x = x[b:b + 1, 4 * hk:4 * hk + 4] if n in ("out", "dq") else x[b:b + 1, hk:hk + 1]
            assert ((x.double().cpu() - ref[n]).abs() <= tol[n]).all(), (n, b, hk)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_largest_values_in_many_workgroups(gpu_device, dtype):
    """Every workgroup, or every other one, goes over its tiles twice: causal means of values near the largest, of equal scores."""
    B, H, N, D = 2, 12, 4100, 64
    g = torch.Generator().manual_seed(7)
    v = ((1.0 + 0.9 * torch.rand(B, H, N, D, generator=g)) * 2.0 ** 127).to(dtype)
    v[:, ::3] *= 2.0 ** -40
    z = torch.zeros(B, H, N, D, dtype=dtype, device=gpu_device)
    for _ in range(5):
        out = window_attention(z, z, v.to(gpu_device), N)
        assert torch.isfinite(out).all()
    want = v.double().cumsum(2) / torch.arange(1, N + 1, dtype=torch.float64)[:, None]
    # Weights are 1; 2 N u of the sums, and the result's half step.
    assert ((out.double().cpu() - want).abs() <= want * (2 * N * 2.0 ** -24 + torch.finfo(dtype).eps / 2 * 1.01)).all()


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("N,window,sinks,at", [(230, 45, 2, 100), (230, 45, 5, 3), (700, 600, 0, 40), (300, 300, 0, 299)])
def test_scores_of_minus_infinity(gpu_device, dtype, N, window, sinks, at):
    """A key with an infinity, against queries whose score it makes -infinity: they give it no weight, and their gradients are those
    of the other keys (but for the infinity's own element, 0 times it)."""
    D = 64
    q, k, v, dout = inputs(1, 1, 1, N, D, dtype)
    q[..., 7] = -q[..., 7].abs() - 0.5
    k[0, 0, at, 7] = torch.inf
    got = run(q, k, v, dout, window, sinks)
    seen = wo.sees(N, window, sinks)
    seen[:, at] = False
    some = seen.any(-1)  # (query 0 or `at` itself may see nothing else)
    x, kk, vv = (t[0, 0].double() for t in (q, k, v))
    kk[at] = 0.0
    x.requires_grad_()
    p = torch.softmax((x @ kk.T * D ** -0.5).masked_fill(~seen, -torch.inf)[some], -1)
    (dq,) = torch.autograd.grad(p @ vv, x, dout[0, 0].double()[some])
    rest = torch.arange(D) != 7
    # As in test_gradients_of_few_keys; float32, which rounds no operand, has its sums' roundings, D for a score.
    bound = torch.finfo(dtype).eps / 2 if dtype != F32 else 2.0 ** -24 * (D * window) ** 0.5
    assert far_off(got["dq"][0, 0][some][:, rest], dq[some][:, rest]) <= bound
    assert far_off(got["out"][0, 0][some], (p @ vv).detach()) <= bound
