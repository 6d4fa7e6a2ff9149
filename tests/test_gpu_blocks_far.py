"""Tensors that reach past 2^31 and 2^32 bytes in the calls with a scale per 128 values, the
RMS norm and the experts' layer: the same bits as from tensors close together, whose
values the other tests check.  And an experts' layer none of whose tokens has an expert."""
import math

import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import Fmt

pytestmark = pytest.mark.gpu

E8 = torch.float8_e8m0fnu


def same(a, b):
    raw = lambda t: t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])
    return torch.equal(raw(a), raw(b))


def far(t, ld):
    """The same values, rows `ld` elements apart."""
    out = torch.empty(t.shape[0] * ld, dtype=t.dtype, device=t.device).view(t.shape[0], ld)[:, :t.shape[1]]
    out.copy_(t)
    assert out.stride(0) * t.shape[0] * t.element_size() > 2 ** 32
    return out


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", [E8, torch.float32])
@pytest.mark.parametrize("M,N,out", [(1100, 2100, torch.bfloat16), (1100, 40, torch.float32)])
def test_products(dev, M, N, out, kind):
    g = torch.Generator(device=dev).manual_seed(1)
    a, sa, _, _ = df.quantize_blocks(torch.randn(M, 500, generator=g, device=dev), scale_dtype=kind)
    b, sb, _, _ = df.quantize_blocks(torch.randn(N, 500, generator=g, device=dev), scale_dtype=kind)
    want = df.gemm_blocks(a, sa, b, sb, 500, out_dtype=out)
    wide = lambda t: far(t.view(torch.uint8), 2 ** 22).view(t.dtype)
    assert same(df.gemm_blocks(wide(a), sa, b, sb, 500, out_dtype=out), want)
    c = torch.empty(M * 2 ** 21, dtype=out, device=dev).view(M, 2 ** 21)[:, :N]
    df.gemm_blocks(a, sa, b, sb, 500, out=c)
    assert same(c, want)
    if N > 1024:
        assert same(df.gemm_blocks(a, sa, wide(b), sb, 500, out_dtype=out), want)


@pytest.mark.parametrize("square", [False, True])
def test_quantizer(dev, square):
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(1100, 300, generator=g, device=dev).bfloat16()
    q = df.quantize_blocks(x, want_qt=True, square=square)
    assert all(same(a, b) for a, b in zip(df.quantize_blocks(far(x, 2 ** 21), want_qt=True, square=square), q))
    rows, cols = 128 * 513, 65536  # codes past 2^32 bytes, both kinds
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    x[:-128] = 1
    x[-128:] = torch.randn(128, cols, generator=g, device=dev)
    q, s, qt, st = df.quantize_blocks(x, Fmt.E4M3, want_qt=True, square=square)
    lq, ls, lqt, lst = df.quantize_blocks(x[-128:].contiguous(), Fmt.E4M3, want_qt=True, square=square)
    assert same(q[-128:], lq) and same(s[:, -128:], ls) and same(qt[:, -128:], lqt) and same(st[-1:], lst)
    assert same(q[:128], q[128:256]) and same(qt[:, :128], qt[:, 128:256])


def test_norm(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev).bfloat16()
    x, r, dy, gamma = rn(1100, 300), rn(1100, 300), rn(1100, 300), rn(300)
    w = [far(t, 2 ** 21) for t in (x, r, dy)]
    for f in (df.rmsnorm_forward, df.rmsnorm_quantize):
        assert all(same(a, b) for a, b in zip(f(w[0], gamma, residual=w[1]), f(x, gamma, residual=r)))
    got, want = (df.rmsnorm_backward(t[2], t[0], gamma, dresidual=t[1]) for t in (w, (x, r, dy)))
    assert same(got[0], want[0]) and same(got[1], want[1])
    del w
    rows, cols = 270000, 16384  # y, the codes and dx past 2^32 bytes
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=dev)
    x[-64:] = rn(64, cols)
    gamma = rn(cols)
    q, s, _, rstd, y = df.rmsnorm_quantize(x, gamma, want_y=True)
    lq, ls, _, lr, ly = df.rmsnorm_quantize(x[-64:].contiguous(), gamma, want_y=True)
    assert same(q[-64:], lq) and same(s[:, -64:], ls) and same(rstd[-64:], lr) and same(y[-64:], ly)
    dx, _ = df.rmsnorm_backward(y, x, gamma, rstd, sums=False)
    ldx, _ = df.rmsnorm_backward(ly, x[-64:].contiguous(), gamma, lr, sums=False)
    assert same(dx[-64:], ldx)


def blocks_of(dev, E, H, N, kind):
    g = torch.Generator(device=dev).manual_seed(4)
    q = lambda *s: df.quantize_experts_blocks(torch.randn(*s, generator=g, device=dev) * s[-1] ** -0.5, scale_dtype=kind)
    return *q(E, 2 * N, H), *q(E, H, N)


@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("kind", [E8, torch.float32])
def test_experts(dev, T, kind):
    E, H, N = 40, 72, 64
    w1, s1, w2, s2 = blocks_of(dev, E, H, N, kind)
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(T, H, generator=g, device=dev).bfloat16()
    logits = torch.randn(T, E, generator=g, device=dev)
    logits[:, -1] += 9  # the last expert's weights are the farthest
    want = df.moe_layer(x, logits, w1, s1, w2, s2, 4)

    def wide(w):
        rows = w.shape[1]
        f = far(w.reshape(E * rows, -1).view(torch.uint8), 2 ** 20 + 2 ** 19).view(w.dtype)
        return f.as_strided(w.shape, (rows * f.stride(0), f.stride(0), 1))

    got = df.moe_layer(x, logits, wide(w1), s1, wide(w2), s2, 4)
    assert all(same(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("T", [1, 2, 64])
@pytest.mark.parametrize("N", [40, 1300])
@pytest.mark.parametrize("none", [-math.inf, math.nan])
def test_no_token_has_an_expert(dev, T, N, none):
    w = blocks_of(dev, 16, 100, N, E8)
    x = torch.full((T, 100), math.nan, dtype=torch.bfloat16, device=dev)
    y, ids, weights = df.moe_layer(x, torch.full((T, 16), none, device=dev), *w, 16)
    assert (y == 0).all() and (ids == -1).all() and (weights == 0).all()
