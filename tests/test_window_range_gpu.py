"""Attention within a window on the GPU at the ends of its range: huge scores, the largest values."""

import pytest
import torch

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
