"""Blocks of 128 values so small that absmax / FMAX rounds to 0 in binary32, and next to
that: every code finite, a zero's code and the codes behind the last value zero, and the
values that codes and scales stand for within the scale's error, for the quantizer and
the norm's codes, and as operands of a product.

Bar: scale and quotient are rounded once each, so a code's value is off by half a step of
the format (or half its least step times the scale) and half a step of binary32's
subnormals times FMAX, from the scale: FMAX * 2^-150.  That covers scale 0 too, where
absmax is below it.
"""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import Fmt

pytestmark = pytest.mark.gpu

E8 = torch.float8_e8m0fnu
FMAX = {Fmt.E4M3: 448.0, Fmt.E5M2: 57344.0}
LEAST = {Fmt.E4M3: 2.0 ** -9, Fmt.E5M2: 2.0 ** -16}
TINY = [1e-45, 1e-44, 1e-43, 3e-43, 4e-43, 1e-42, 3e-41, 4e-41, 5e-41, 1e-40, 1e-38]


def check(x, q, s, fmt):
    """x [R, C] binary64 on the device, its codes and scales."""
    R, C = x.shape
    raw = q.view(torch.uint8)
    assert q.float().isfinite().all() and s.float().isfinite().all()
    assert not raw[:, C:].any() and not (raw[:, :C][x == 0] & 0x7F).any()
    step = s.double().t().repeat_interleave(128, 1)[:, :C]
    bar = torch.maximum(torch.finfo(q.dtype).eps / 2 * x.abs(), LEAST[fmt] / 2 * step) + FMAX[fmt] * 2.0 ** -150
    assert ((q[:, :C].double() * step - x).abs() <= bar).all()


def mixed(dev, R, C, seed=0):
    """Rows of values up to a tiny one, half of them zero, some of either sign."""
    g = torch.Generator(device=dev).manual_seed(seed)
    top = torch.tensor(TINY, device=dev, dtype=torch.float64)[torch.arange(R, device=dev) % len(TINY)]
    x = top[:, None] * torch.randn(R, C, generator=g, device=dev).clamp(-1, 1)
    return torch.where(torch.rand(R, C, generator=g, device=dev) < 0.5, x, 0.0).float()


@pytest.mark.parametrize("fmt", list(Fmt))
@pytest.mark.parametrize("kind", [E8, torch.float32])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("R,C", [(1, 1), (11, 7), (13, 130), (200, 333)])
def test_quantizer(dev, kind, fmt, square, R, C):
    x = mixed(dev, R, C)
    for t in (x, x.t().contiguous(), torch.where(x.abs() < 1e-44, x, 0.0)):
        q, s, qt, st = df.quantize_blocks(t, fmt, want_qt=True, square=square, scale_dtype=kind)
        check(t.double(), q, s, fmt)
        check(t.t().double(), qt, st, fmt)


@pytest.mark.parametrize("kind", [E8, torch.float32])
def test_nan_and_infinity_among_tiny_values(dev, kind):
    x = mixed(dev, 22, 140)
    x[3, 5], x[4, 6], x[1, 139] = float("nan"), float("inf"), -float("nan")
    q, s, _, _ = df.quantize_blocks(x, scale_dtype=kind)
    raw = q.view(torch.uint8)
    assert raw[3, 5] == 0x7F and raw[1, 139] == 0xFF and raw[4, 6] == 0x7E
    assert torch.equal(q.float().isnan().nonzero(), torch.tensor([[1, 139], [3, 5]], device=dev))


@pytest.mark.parametrize("fmt", list(Fmt))
@pytest.mark.parametrize("kind", [E8, torch.float32])
@pytest.mark.parametrize("cols", [7, 200, 1600, 5001, 20001])
def test_norm(dev, kind, fmt, cols):
    """gamma of tiny values and zeros."""
    g = torch.Generator(device=dev).manual_seed(cols)
    x = torch.randn(5, cols, generator=g, device=dev)
    for top in (1e-45, 1e-44, 2e-43, 1e-41, 1e-39):
        gamma = torch.where(torch.rand(cols, generator=g, device=dev) < 0.5, top, 0.0)
        q, s, _, _, y = df.rmsnorm_quantize(x, gamma, fmt=fmt, want_y=True, scale_dtype=kind)
        check(y.double(), q, s, fmt)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(20, 40, 300), (700, 600, 300)])
def test_product_of_a_tiny_gradient(dev, out, M, N, K):
    """Nothing but zeros and values next to binary32's least: the product is next to 0,
    and no row or column of it is lost."""
    a, sa, _, _ = df.quantize_blocks(mixed(dev, M, K), Fmt.E5M2, scale_dtype=torch.float32)
    b, sb, _, _ = df.quantize_blocks(torch.randn(N, K, device=dev), scale_dtype=torch.float32)
    c = df.gemm_blocks(a, sa, b, sb, K, out_dtype=out)
    assert c.isfinite().all() and c.abs().max() < 1e-34
