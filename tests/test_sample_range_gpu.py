"""Sampling on the GPU at the ends of its range: more rows than one grid holds."""

import pytest
import torch

from dwarf_amd import sample_tokens

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
