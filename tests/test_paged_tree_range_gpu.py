"""Drafted-token steps on the GPU at the ends of their range: huge scores."""

import pytest
import torch

from dwarf_amd import paged_tree_step
from oracle import paged_oracle as po
from tests.test_paged_gpu import Cache
from tests.test_paged_tree_gpu import BF, E4, F16, F32, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,kv", [(F16, F16), (F16, E4), (BF, BF), (F32, F32)])
@pytest.mark.parametrize("T", [8, 30])
@pytest.mark.parametrize("power", [14, 20, 22, 23, 24, 25, 26, 28])
def test_huge_scores(gpu_device, dtype, kv, T, power):
    """Scores up to 2^40 give the row of the largest.  Sums of |q||k| are below 2^12, so that a score is off by 40 2^-12 times
    the scale at most, and one that is ahead by 2^8 besides leaves the others exp(-2^8) of its weight: nothing.  What is left of
    the row is its weight's two 16-bit terms, 2^-16 of it, or one that is exact, and a half step of the output."""
    D, pos = 32, [200, 31, 0, 77]
    c = Cache(gpu_device, 4, 1, D, 16, 16, dtype, kv, [p + T for p in pos])
    g = torch.Generator().manual_seed(power)
    q, k, v = (torch.randn(4, 1, T, D, generator=g).to(dtype).to(gpu_device) for _ in range(3))
    parents = [tree(T, b) for b in range(4)]
    out = paged_tree_step(q, k, v, c.k, c.v, c.table, torch.tensor(pos, device=gpu_device), torch.tensor(parents, device=gpu_device),
                          softmax_scale=2.0 ** power, **c.state).double().cpu()
    sure = 0
    for b, n in enumerate(pos):
        nodes = po.tree_rows(parents[b], T)
        kk, vv = c.rows("k", b, n + T)[0], c.rows("v", b, n + T)[0]
        for i, node in enumerate(nodes):
            sees = po.tree_sees(node, nodes, n)
            x = q[b, 0, i].double().cpu()
            assert torch.isfinite(out[b, 0, i]).all(), (b, i)
            assert (kk[sees].abs() @ x.abs()).max() < 2 ** 12
            s = torch.cat([kk[sees] @ x, torch.tensor([-torch.inf], dtype=torch.float64)])
            first, second = s.topk(2).values.tolist()
            if first - second > 2 * 40 * 2.0 ** -12 + 2.0 ** (8 - power):
                sure += 1
                want = vv[sees[int(s.argmax())]]
                assert ((out[b, 0, i] - want).abs() <= want.abs() * (2.0 ** -16 + torch.finfo(dtype).eps / 2)).all(), (b, i)
    assert sure > 3 * T
