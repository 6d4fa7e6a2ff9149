"""The norm of 2-byte gradients over their whole range, and a clipped step on it."""
import numpy as np
import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e25), (torch.bfloat16, 1e34), (torch.bfloat16, 1e-25),
                                        (torch.bfloat16, 1e-37), (torch.float16, 6e4), (torch.float16, 6e-8)])
@pytest.mark.parametrize("n", [5, 8192, 40_001])
def test_norm_of_large_and_small(dev, dtype, size, n):
    g = torch.Generator(device=dev).manual_seed(n)
    x = ((torch.rand(n, generator=g, device=dev) * 2 - 1) * size).to(dtype)
    want = x.double().square().sum().sqrt().item()
    # exact squares, a binary64 sum of n terms, one rounding of the root to binary32
    assert abs(df.grad_norm([x]).item() - want) <= (2.0 ** -24 + n * 2.0 ** -53) * want


def test_clipped_step_of_large_gradients(dev):
    """A gradient of 1e20 is clipped to max_norm, not lost: the first step moves by lr along its sign."""
    p, g = torch.zeros(300, device=dev), torch.full((300,), 1e20, dtype=torch.bfloat16, device=dev)
    g[::2] *= -1
    ms, vs, _, _ = df.adamw_state([p])
    df.adamw_update([p], [g], ms, vs, 1, lr=1e-2, weight_decay=0.0, clip_norm=df.grad_norm([g]), max_norm=1.0)
    # m / sqrt(v) is 1 but for a few roundings (6 of 2^-24) and eps = 1e-8 beside 1 / sqrt(300) (2e-7)
    assert np.allclose(p.cpu().numpy() * np.sign(-g.float().cpu().numpy()), 1e-2, rtol=1e-6, atol=0)
