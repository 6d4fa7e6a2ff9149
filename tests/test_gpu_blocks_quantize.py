"""df_quantize_blocks against its rule on the CPU, bit for bit: scales and codes,
row and transposed, per 128 and per 128 x 128, at sizes around a block's edges,
strides, alignments, and values that are zero, tiny, huge, infinite or NaN.

No tolerance: a power-of-two scale divides exactly and an fp32 one by IEEE
division, and one rounding to the format follows.
"""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import Fmt

pytestmark = pytest.mark.gpu

E8 = torch.float8_e8m0fnu
FMAX = {Fmt.E4M3: 448.0, Fmt.E5M2: 57344.0}
CODE = {Fmt.E4M3: torch.float8_e4m3fn, Fmt.E5M2: torch.float8_e5m2}


def finite_absmax(x, dim):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dim)


def scale_of(most, fmt, dtype):
    """The rule in 64 bits; [..] fp32 values."""
    if dtype == torch.float32:
        return torch.where(most > 0, most / torch.tensor(FMAX[fmt]), torch.ones_like(most))
    m = most.double()
    e = torch.ceil(torch.log2(torch.where(m > 0, m, torch.ones_like(m)) / FMAX[fmt]))
    e = torch.where(2.0 ** (e - 1) * FMAX[fmt] >= m, e - 1, e)  # log2 rounded up at a power of two
    e = torch.where(2.0 ** e * FMAX[fmt] < m, e + 1, e)
    return torch.where(m > 0, 2.0 ** e.clamp(min=-127), torch.ones_like(m)).float()


def codes_of(x, s, fmt):
    q = (x / s).clamp(-FMAX[fmt], FMAX[fmt]).to(CODE[fmt]).view(torch.uint8)
    nan = torch.where(torch.signbit(x), 0xFF, 0x7F).to(torch.uint8)
    return torch.where(torch.isnan(x), nan, q)


def rows_rule(x, fmt, dtype, square):
    """(codes [R, ceil16(C)], scales [blocks, R]) of fp32 x on the CPU."""
    R, C = x.shape
    nb = -(-C // 128)
    pad = torch.zeros(-(-R // 128) * 128, nb * 128)
    pad[:R, :C] = x
    most = finite_absmax(pad.view(-1, nb, 128), 2)
    if square:
        most = most.view(-1, 128, nb).amax(1).repeat_interleave(128, 0)
    s = scale_of(most[:R], fmt, dtype)
    q = codes_of(pad[:R].view(R, nb, 128), s[:, :, None], fmt).view(R, -1)
    return q[:, :-(-C // 16) * 16], s.t()


def check(x, fmt, dtype, square, want_q=True, want_qt=True):
    q, s, qt, st = df.quantize_blocks(x, fmt, want_q=want_q, want_qt=want_qt, square=square, scale_dtype=dtype)
    host = x.float().cpu()
    for want, codes, scales, m in ((want_q, q, s, host), (want_qt, qt, st, host.t().contiguous())):
        if not want:
            assert codes is None and scales is None
            continue
        rq, rs = rows_rule(m, fmt, dtype, square)
        assert scales.dtype == dtype and torch.equal(scales.float().cpu(), rs)
        assert codes.dtype == CODE[fmt] and torch.equal(codes.view(torch.uint8).cpu(), rq)


def data(dev, R, C, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(R, C, generator=g, device=dev) * torch.exp(3 * torch.randn(R, 1, generator=g, device=dev))
    return (x * torch.exp(torch.randn(1, C, generator=g, device=dev))).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scales", [E8, torch.float32])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 768), (3, 7), (8, 9), (16, 128), (127, 129), (128, 128), (130, 1600), (771, 257)])
def test_sizes(dev, dtype, scales, square, R, C):
    for fmt in Fmt:
        check(data(dev, R, C, dtype), fmt, scales, square)


@pytest.mark.parametrize("want", [(True, False), (False, True)])
def test_one_kind_of_codes(dev, want):
    check(data(dev, 200, 300, torch.bfloat16), Fmt.E4M3, E8, False, *want)
    check(data(dev, 200, 300, torch.bfloat16), Fmt.E5M2, torch.float32, True, *want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("off,pad", [(1, 0), (3, 5), (0, 13)])
def test_any_address_and_stride(dev, dtype, off, pad):
    wide = data(dev, 140, off + 333 + pad, dtype)
    check(wide[:, off:off + 333], Fmt.E4M3, E8, False)
    check(wide.reshape(-1)[off:off + 140 * 200].view(140, 200), Fmt.E4M3, torch.float32, False)


@pytest.mark.parametrize("scales", [E8, torch.float32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("square", [False, True])
def test_special_values(dev, dtype, scales, square):
    x = data(dev, 300, 400, torch.float32).clamp(-6e4, 6e4)
    x[0] = 0.0
    x[1, ::2] = -0.0
    x[2, 130] = float("inf")
    x[3, 5] = -float("inf")
    x[4, 7], x[4, 8] = float("nan"), -float("nan")
    x[5] = float("nan")
    x[6] = float("inf")
    x[128:256, 128:256] = 0.0
    x[7, :128] = 448.0
    x[7, 128:256] = 448.0 * 2 ** -10
    x[8, :128] = 57344.0
    x[9, 0] = 449.0
    if dtype == torch.float32:
        x[10] = 1e-38
        x[11] = 1e-44
        x[12] = 3e38
    elif dtype == torch.float16:
        x[10] = 6e-8
    for fmt in Fmt:
        check(x.to(dtype), fmt, scales, square)


def test_no_rows_or_columns(dev):
    for R, C in ((0, 5), (5, 0), (0, 0)):
        q, s, qt, st = df.quantize_blocks(torch.empty(R, C, device=dev), want_qt=True)
        assert q.shape == (R, -(-C // 16) * 16) and s.shape == (-(-C // 128), R)
        assert qt.shape == (C, -(-R // 16) * 16) and st.shape == (-(-R // 128), C)


@pytest.mark.parametrize("dtype", [E8, torch.float32])
def test_block_scales(dev, dtype):
    s = torch.exp2(torch.randint(-20, 20, (5, 3), device=dev).float()).to(dtype)
    got = df.block_scales(s)
    assert got.shape == (3, 5) and got.dtype == dtype and torch.equal(got.float(), s.float().t())
    assert got.stride(0) * dtype.itemsize % 16 == 0
    got = df.block_scales(s, rows=600)
    assert got.shape == (3, 600) and torch.equal(got.float(), s.float().t().repeat_interleave(128, 1)[:, :600])
