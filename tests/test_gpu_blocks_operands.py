"""Operands of the calls with a scale per 128 values that end where their last row's
codes do, or have other values next to them: the same bits as from tensors of their own."""
import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu

E8 = torch.float8_e8m0fnu


def same(a, b):
    raw = lambda t: t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])
    return torch.equal(raw(a), raw(b))


def right_half(w, side):
    """w's codes as the columns from `side` on of a matrix whose others are NaN; the last
    row's leading dimension reaches `side` bytes past the storage."""
    E, R, C = w.shape
    wide = torch.full((E, R, side + C), 0x7F, dtype=torch.uint8, device=w.device).view(w.dtype)
    wide[:, :, side:].view(torch.uint8).copy_(w.view(torch.uint8))
    return wide[:, :, side:]


@pytest.mark.parametrize("T", [1, 2, 40])
@pytest.mark.parametrize("H,N", [(40, 24), (300, 130), (16, 16)])
@pytest.mark.parametrize("side", [16, 400])
def test_experts_weights_beside_others(dev, T, H, N, side):
    g = torch.Generator(device=dev).manual_seed(T)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)
    w1, s1 = df.quantize_experts_blocks(n(5, 2 * N, H))
    w2, s2 = df.quantize_experts_blocks(n(5, H, N))
    x, logits = n(T, H).bfloat16(), n(T, 5)
    logits[:, 4] += 9  # the last expert's last rows
    want = df.moe_layer(x, logits, w1, s1, w2, s2, 2)
    got = df.moe_layer(x, logits, right_half(w1, side), s1, right_half(w2, side), s2, 2)
    assert all(same(a, b) for a, b in zip(got, want)) and got[0].isfinite().all()


@pytest.mark.parametrize("kind", [E8, torch.float32])
@pytest.mark.parametrize("K", [40, 771])
def test_products_of_one_row(dev, kind, K):
    """One row of a packed matrix of padded rows; one whose memory ends with its codes."""
    g = torch.Generator(device=dev).manual_seed(K)
    a, sa, _, _ = df.quantize_blocks(torch.randn(5, K, generator=g, device=dev), scale_dtype=kind)
    b, sb, _, _ = df.quantize_blocks(torch.randn(70, K, generator=g, device=dev), scale_dtype=kind)
    want = df.gemm_blocks(a, sa, b, sb, K)
    for r in (0, 4):
        s = df.block_scales(sa[:, r:r + 1].t())
        assert same(df.gemm_blocks(a[r:r + 1, :K], s, b, sb, K), want[r:r + 1])
        one = a[r:r + 1].clone()
        assert same(df.gemm_blocks(one, s, b, sb, K), want[r:r + 1])
