"""Attention within a window on the GPU at the ends of its range: huge scores."""

import pytest
import torch

from oracle import window_oracle as wo
from tests.test_window_gpu import BF, F16, F32, inputs, run

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
