"""Products with fp32 scales per 128 whose size, or whose neighbours in memory, are
unusual: scales whose product with each other or with a step's sum leaves binary32's
range though the result does not, zero scales, and values behind the last column.

Bars as in test_gpu_blocks_gemm.py; a result below binary32's normal range adds its
step, 2^-149, once for each of K / 128 blocks and eight waves.
"""
import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu

E4 = torch.float8_e4m3fn
U32 = torch.finfo(torch.float32).eps / 2
# small tiles of every kind, 128 x 128, 256 x 128
SIZES = [(3, 37, 300), (16, 5003, 300), (70, 1601, 300), (300, 771, 515), (1030, 1603, 700), (4100, 1603, 399)]


def codes(g, rows, K, lo, hi, dev):
    q = torch.zeros(rows, -(-K // 16) * 16, dtype=torch.uint8, device=dev)
    mag = torch.randint(lo, hi + 1, (rows, K), generator=g, device=dev)
    q[:, :K] = (mag + 128 * torch.randint(0, 2, (rows, K), generator=g, device=dev)).to(torch.uint8)
    return q.view(E4)


def scales(g, blocks, rows, exponent, dev, square):
    """[blocks, rows] near 2^exponent; square: one for 128 rows."""
    s = 1 + torch.rand(-(-rows // 128) if square else rows, blocks, generator=g, device=dev, dtype=torch.float64)
    return df.block_scales((s * 2.0 ** exponent).float(), rows if square else None)


def values(q, s, K):
    return q[:, :K].double() * s.double().t().repeat_interleave(128, 1)[:, :K]


def check(got, a, sa, b, sb, K):
    va, vb = values(a, sa, K), values(b, sb, K)
    want, size = va @ vb.t(), va.abs() @ vb.abs().t()
    if got.dtype == torch.float32:
        bar = (K + 64) * U32 * size + (K / 128 + 9) * 2.0 ** -149
    else:
        bar = torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0 ** -10 * size + torch.finfo(got.dtype).smallest_normal
    assert want.abs().max() < 2.0 ** 126  # (no result is near the type's end)
    assert ((got.double() - want).abs() <= bar).all()


@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_far_scales(dev, out, square, M, N, K):
    g = torch.Generator(device=dev).manual_seed(M)
    nb = -(-K // 128)
    # large codes: sums near 2^20; small ones: near 2^-10
    for lo, hi, ea, eb in ((0x70, 0x7E, -120, -20), (0x70, 0x7E, -20, -120), (0x70, 0x7E, -110, 112), (0x70, 0x7E, 112, -110),
                           (1, 4, 66, 64), (1, 16, 120, -122), (1, 16, -122, 120), (0x70, 0x7E, -140, 60), (0x70, 0x7E, 60, -140)):
        a, b = codes(g, M, K, lo, hi, dev), codes(g, N, K, lo, hi, dev)
        sa, sb = scales(g, nb, M, ea, dev, False), scales(g, nb, N, eb, dev, square)
        check(df.gemm_blocks(a, sa, b, sb, K, out_dtype=out), a, sa, b, sb, K)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_far_scales_among_others(dev, out, M, N, K):
    """Some far, some zero, most of them ordinary; blocks of zero codes at scales whose
    product is infinite."""
    g = torch.Generator(device=dev).manual_seed(N)
    nb = -(-K // 128)
    a, b = codes(g, M, K, 0x30, 0x48, dev), codes(g, N, K, 0x30, 0x48, dev)
    sa, sb = scales(g, nb, M, 0, dev, False), scales(g, nb, N, -10, dev, False)
    sa[0, M // 2], sa[nb - 1, M - 1], sa[1, 0] = 2.0 ** -110, 2.0 ** 70, 0.0
    sb[0, N // 3], sb[1, N - 1], sb[nb - 1, 1] = 2.0 ** -115, 2.0 ** -149, 0.0
    a.view(torch.uint8)[M // 2, 128:256], sa[1, M // 2] = 0, 2.0 ** 100
    b.view(torch.uint8)[2, 128:256], sb[1, 2] = 0, 2.0 ** 100
    check(df.gemm_blocks(a, sa, b, sb, K, out_dtype=out), a, sa, b, sb, K)


@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES + [(2000, 1000, 500), (8200, 1100, 300)])
def test_values_behind_the_scales_change_nothing(dev, out, square, M, N, K):
    """Scales' rows are padded with whatever the memory held: the same bits."""
    g = torch.Generator(device=dev).manual_seed(K)
    nb = -(-K // 128)
    a, b = codes(g, M, K, 0x18, 0x48, dev), codes(g, N, K, 0x18, 0x48, dev)
    sa, sb = scales(g, nb, M, -3, dev, False), scales(g, nb, N, -5, dev, square)

    def padded(s, fill):
        wide = torch.full((nb, -(-s.shape[1] // 4) * 4 + 256), float(fill), device=dev)
        wide[:, :s.shape[1]] = s
        if fill == 0:  # the last one's, as if they went on
            wide[:, s.shape[1]:] = s[:, -1:]
        return wide[:, :s.shape[1]]

    first = df.gemm_blocks(a, padded(sa, 0), b, padded(sb, 0), K, out_dtype=out)
    check(first, a, sa, b, sb, K)
    raw = torch.int32 if out == torch.float32 else torch.int16
    for fill in (1.0, float("nan"), float("inf"), 2.0 ** -140, 2.0 ** 120):
        got = df.gemm_blocks(a, padded(sa, fill), b, padded(sb, fill), K, out_dtype=out)
        assert torch.equal(got.view(raw), first.view(raw))
