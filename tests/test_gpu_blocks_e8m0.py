"""Power-of-two scales at the ends of their range, 2^-127 (byte 0) to 2^127 (byte 254),
where the result is ordinary: the products at codes whose values bf16 holds (fp32 outputs
go through it: multiples of 2^-133 below 2^128, so codes from 2^-3 on at 2^-127), the
experts' layer likewise in W2.  Bars as in test_gpu_blocks_gemm.py and test_gpu_moe.py."""
import pytest
import torch

import deepfuse_amd as df
from test_gpu_blocks_gemm import E4, E5, E8, check
from test_gpu_moe import check as check_layer

pytestmark = pytest.mark.gpu

SIZES = [(5, 40, 300), (13, 4201, 300), (70, 1601, 300), (569, 1317, 645), (700, 1603, 1100), (923, 2193, 300), (2045, 4595, 515)]


def codes(g, rows, K, lo, hi, dtype, dev):
    q = torch.zeros(rows, -(-K // 16) * 16, dtype=torch.uint8, device=dev)
    mag = torch.randint(lo, hi + 1, (rows, K), generator=g, device=dev)
    q[:, :K] = (mag + 128 * torch.randint(0, 2, (rows, K), generator=g, device=dev)).to(torch.uint8)
    return q.view(dtype)


def scales(g, blocks, rows, lo, hi, dev):
    """Bytes lo to hi."""
    return df.block_scales(torch.randint(lo, hi + 1, (rows, blocks), generator=g, device=dev).to(torch.uint8).view(E8))


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_products(dev, out, M, N, K):
    g = torch.Generator(device=dev).manual_seed(M)
    nb = -(-K // 128)
    # codes of 2^-3 and more at the least scales, below 2 at the largest ones
    for fa, lo, hi in ((E4, 0x20, 0x3F), (E5, 0x30, 0x3F)):
        for (a0, a1), (b0, b1) in (((0, 3), (240, 246)), ((240, 246), (0, 3)), ((0, 1), (250, 254)), ((250, 254), (0, 1)),
                                   ((0, 2), (252, 254)), ((120, 134), (120, 134))):
            a, b = codes(g, M, K, lo, hi, fa, dev), codes(g, N, K, 0x20, 0x3F, E4, dev)
            sa, sb = scales(g, nb, M, a0, a1, dev), scales(g, nb, N, b0, b1, dev)
            check(df.gemm_blocks(a, sa, b, sb, K, out_dtype=out), a, sa, b, sb, K)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_layer(dev, T):
    """W2 at 2^-127 and next to it, inner values near 2^100."""
    g = torch.Generator(device=dev).manual_seed(T)
    E, H, N = 4, 200, 300
    w1 = codes(g, E * N, H, 0x20, 0x3F, E4, dev).view(E, N, -1)
    w2 = codes(g, E * H, N, 0x20, 0x3F, E4, dev).view(E, H, -1)
    s = lambda rows, cols, lo, hi: torch.randint(lo, hi, (E, -(-cols // 128), -(-rows // 16) * 16), generator=g,
                                                 device=dev).to(torch.uint8).view(E8)[:, :, :rows]
    s1, s2 = s(N, H, 215, 220), s(H, N, 0, 4)
    x = torch.randn(T, H, generator=g, device=dev).bfloat16()
    logits = torch.randn(T, E, generator=g, device=dev)
    out = df.moe_layer(x, logits, w1, s1, w2, s2, 2, activation="gelu")
    assert out[0].abs().max() > 2.0 ** -40
    check_layer(out, x, logits, w1, s1, w2, s2, 2, "gelu")


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_bytes_behind_the_scales_change_nothing(dev, out, M, N, K):
    """Scales' rows are padded with whatever the memory held, NaN's byte too."""
    g = torch.Generator(device=dev).manual_seed(K)
    nb = -(-K // 128)
    a, b = codes(g, M, K, 0x20, 0x47, E4, dev), codes(g, N, K, 0x20, 0x47, E4, dev)
    sa, sb = scales(g, nb, M, 110, 130, dev), scales(g, nb, N, 110, 130, dev)

    def padded(s, fill):
        wide = torch.full((nb, -(-s.shape[1] // 16) * 16 + 256), fill, dtype=torch.uint8, device=dev)
        wide[:, :s.shape[1]] = s.view(torch.uint8)
        return wide.view(E8)[:, :s.shape[1]]

    raw = torch.int32 if out == torch.float32 else torch.int16
    first = df.gemm_blocks(a, padded(sa, 127), b, padded(sb, 127), K, out_dtype=out)
    check(first, a, sa, b, sb, K)
    for fill in (0, 254, 255):
        got = df.gemm_blocks(a, padded(sa, fill), b, padded(sb, fill), K, out_dtype=out)
        assert torch.equal(got.view(raw), first.view(raw))
