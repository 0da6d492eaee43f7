"""Sampling on the GPU at the ends of its range: more rows than one grid holds, long rows by one workgroup each, rows whose
stretches are longer than 64 pieces."""

import math

import pytest
import torch

from dwarf_amd import sample_tokens
from oracle import sample_oracle as so
from tests.test_sample_gpu import BF, F16, F32, check, rows

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_grid_holds(gpu_device):
    """2^22 + 3 rows of 1024 lanes each: the same as in calls of their own, with settings of each row."""
    B, V, dev = (1 << 22) + 3, 5, gpu_device
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(B, V + 1, generator=g, device=dev).to(torch.bfloat16)[:, 1:]
    u = torch.rand(B, generator=g, device=dev, dtype=torch.float64)
    t, p, m = (torch.rand(B, generator=g, device=dev) for _ in range(3))
    k = torch.randint(0, V + 1, (B,), generator=g, device=dev)
    for settings in ((t, k, p, m * 0.3), (0.8, 0, 0.9, 0.0)):
        tokens, logp = sample_tokens(x, u, *settings, return_logprobs=True)
        for rows in (slice(0, 1000), slice((1 << 21) - 500, (1 << 21) + 500), slice((1 << 22) - 500, B)):
            a, b = sample_tokens(x[rows], u[rows], *(s[rows] if torch.is_tensor(s) else s for s in settings), return_logprobs=True)
            assert torch.equal(tokens[rows], a) and torch.equal(logp[rows], b)
        assert ((tokens >= 0) & (tokens < V)).all() and (logp <= 0).all()


@pytest.mark.parametrize("V,dtype", [(8193, F32), (32000, BF), (33333, F16)])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, top_p=0.8), dict(top_p=0.9, min_p=1e-3), dict(top_k=1500), dict(top_p=0.9999),
                                dict(temperature=0.0)])
def test_a_workgroup_for_a_long_row(gpu_device, V, dtype, kw):
    """Batches of 129 rows and more are not split: each workgroup goes over its row several times round.  Some rows against the
    oracle, and all of them against calls of a few, whose rows several workgroups share: masses are whole numbers, so that the
    results are the same."""
    x, u = rows(131, V + 1, V, dtype)
    x = x[:, 1:]
    x[1] = 0.25
    x[2, torch.arange(V) % 997 != 5] = -math.inf
    kw = {"temperature": 0.8, **kw}
    xd, ud = x.to(gpu_device), u.to(gpu_device)
    tokens, logp = sample_tokens(xd, ud, **kw, return_logprobs=True)
    for b in range(0, 131, 10):
        t, lp = sample_tokens(xd[b:b + 10], ud[b:b + 10], **kw, return_logprobs=True)
        assert torch.equal(tokens[b:b + 10], t) and torch.equal(logp[b:b + 10], lp)
    tol = V * 2.0 ** -(48 if V <= 1 << 14 else 62 - (V - 1).bit_length())
    sure = 0
    for b in (0, 1, 2, 77, 130):
        t, lp, margin = so.sample(x[b].double().tolist(), u[b].item(), **kw)
        if margin > tol:
            sure += 1
            # (As in check: half a step of float32, and the masses' rounding.)
            assert tokens[b] == t and (logp[b] == lp or abs(logp[b].item() - lp) <= 2.0 ** -24 * abs(lp) + 2 * tol), b
    assert sure >= 3


@pytest.mark.parametrize("V,dtype", [(600001, BF), (530000, F32)])
def test_long_stretches(gpu_device, V, dtype):
    """Above 2^19 tokens the last sum's stretches are longer than 64 pieces."""
    x, u = rows(4, V, 5, dtype)
    x[3] = 1.5
    for kw in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.7), dict(temperature=0.0)):
        check(x, u, **kw)
    # By one workgroup each: as split.
    many = x.to(gpu_device).repeat(40, 1)
    for kw in (dict(), dict(top_k=40), dict(top_p=0.7)):
        a = sample_tokens(x.to(gpu_device), u.to(gpu_device), **kw, return_logprobs=True)
        b = sample_tokens(many, u.to(gpu_device).repeat(40), **kw, return_logprobs=True)
        assert torch.equal(a[0].repeat(40), b[0]) and torch.equal(a[1].repeat(40), b[1])
