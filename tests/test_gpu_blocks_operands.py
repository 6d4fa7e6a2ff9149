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


@pytest.mark.parametrize("kind", [E8, torch.float32])
def test_a_batch_of_no_tokens(dev, kind):
    """A training step's calls: outputs without rows, gradients of the weights zero."""
    K, N = 300, 200
    g = torch.Generator(device=dev).manual_seed(0)
    x, w, dy = torch.empty(0, K, device=dev), torch.randn(N, K, generator=g, device=dev), torch.empty(0, N, device=dev)
    gamma = torch.ones(K, device=dev)
    xq, sx, s, rstd, y = df.rmsnorm_quantize(x, gamma, want_y=True, scale_dtype=kind)
    wq, sw, wt, swt = df.quantize_blocks(w, want_qt=True, square=True, scale_dtype=kind)
    assert df.gemm_blocks(xq, sx, wq, sw, K).shape == (0, N)
    xq, sx, xt, sxt = df.quantize_blocks(y, want_qt=True, scale_dtype=kind)
    dyq, sdy, dyt, sdyt = df.quantize_blocks(dy, df.Fmt.E5M2, want_qt=True, scale_dtype=kind)
    assert df.gemm_blocks(xq, sx, wq, sw, K).shape == (0, N)
    dx = df.gemm_blocks(dyq, sdy, wt, swt, N, out_dtype=torch.float32)
    assert dx.shape == (0, K)
    dw = df.gemm_blocks(dyt, sdyt, xt, sxt, 0, out_dtype=torch.float32)
    assert dw.shape == (N, K) and not dw.any()
    dx, dg = df.rmsnorm_backward(dx, s, gamma, rstd)
    assert dx.shape == (0, K) and not dg.any()
