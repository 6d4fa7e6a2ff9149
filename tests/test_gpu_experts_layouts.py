"""The experts' products on codes with a dimension of one, whose stride is
arbitrary: weights of one output column, one row, transposed and cut views, each
equal to the call on a plain copy and to the product in binary64."""
import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def codes(g, dev, shape, fmt):
    """codes of small whole numbers: sums of their products are exact in binary32"""
    return torch.randint(-8, 9, shape, generator=g, device=dev).float().to(fmt).view(torch.uint8)


def one_column(w):
    """the codes [E, 1, K] in every layout with the experts a fixed step apart"""
    E, K = w.shape
    wide = torch.full((E, 3, K + 32), 0x7F, dtype=torch.uint8, device=w.device)
    wide[:, 1, :K] = w
    return [w[:, None], w[None].transpose(0, 1), wide[:, 1:2, :K], w.clone().as_strided((E, 1, K), (K, 16, 1))]


@pytest.mark.parametrize("which", ["fwd", "dx"])
@pytest.mark.parametrize("E,K,counts", [(4, 32, [3, 0, 40, 1]), (3, 1600, [700, 900, 20])])
def test_one_column(dev, which, E, K, counts):
    g = torch.Generator(device=dev).manual_seed(K)
    fmt, fn = (E4, df.experts_fwd) if which == "fwd" else (E5, df.experts_dx)
    b = [0]
    for c in counts:
        b.append(b[-1] + c)
    x, w = codes(g, dev, (b[-1], K), fmt), codes(g, dev, (E, K), E4)
    off, s = torch.tensor(b, dtype=torch.int32, device=dev), torch.ones(1, device=dev)
    sw = 2.0 ** -torch.arange(E, device=dev).float()
    ref = torch.cat([x[lo:hi].view(fmt).double() @ w[e].view(E4).double()[:, None] * sw[e].double()
                     for e, (lo, hi) in enumerate(zip(b, b[1:]))])
    for v in one_column(w):
        for dt in (torch.float32, torch.bfloat16):
            assert torch.equal(fn(x, v, off, K, s, sw, out_dtype=dt), ref.to(dt)), v.stride()


def one_row(r):
    K = r.shape[0]
    wide = torch.full((3, K + 48), 0x7F, dtype=torch.uint8, device=r.device)
    wide[1, :K] = r
    return [r[None], r[:, None].t(), wide[1:2, :K], r.clone().as_strided((1, K), (5, 1))]


@pytest.mark.parametrize("K,N", [(32, 48), (1600, 2112)])
def test_one_row(dev, K, N):
    g = torch.Generator(device=dev).manual_seed(N)
    off, s, sw = torch.tensor([0, 0, 1], dtype=torch.int32, device=dev), torch.ones(1, device=dev), torch.ones(2, device=dev)
    w = codes(g, dev, (2, N, K), E4)
    for fn, fmt in ((df.experts_fwd, E4), (df.experts_dx, E5)):
        x = codes(g, dev, (K,), fmt)
        ref = (x.view(fmt).double() @ w[1].view(E4).double().t()).float()
        for v in one_row(x):
            assert torch.equal(fn(v, w, off, K, s, sw, out_dtype=torch.float32)[0], ref), v.stride()


def test_one_row_dw(dev):
    """dW of one output or one input: the transposed codes are one row."""
    g = torch.Generator(device=dev).manual_seed(7)
    R, M = 64, 40
    off, s = torch.tensor([0, 30, 61], dtype=torch.int32, device=dev), torch.ones(1, device=dev)
    many = {f: codes(g, dev, (M, R), f) for f in (E4, E5)}
    one = {f: codes(g, dev, (R,), f) for f in (E4, E5)}
    d = lambda t, f: t.view(f).double()
    for e5, e4 in zip(one_row(one[E5]), one_row(one[E4])):
        a, b = df.experts_dw(e5, many[E4], off, R, s, s), df.experts_dw(many[E5], e4, off, R, s, s)
        for e, (lo, hi) in enumerate(((0, 30), (30, 61))):
            assert torch.equal(a[e, 0].double(), d(many[E4], E4)[:, lo:hi] @ d(one[E5], E5)[lo:hi])
            assert torch.equal(b[e, :, 0].double(), d(many[E5], E5)[:, lo:hi] @ d(one[E4], E4)[lo:hi])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,N,K", [(3, 40, 96), (5, 37, 51), (1, 16, 16)])
def test_quantize_weights_at_any_element(dev, dtype, E, N, K):
    g = torch.Generator(device=dev).manual_seed(E)
    w = torch.randn(E, N, K, generator=g, device=dev).to(dtype)
    want = df.quantize_experts(w)
    for off in (1, 3, 8):
        base = torch.full((E * N * K + 16,), 1e4, device=dev).to(dtype)
        view = base[off:off + E * N * K].view(E, N, K)
        view.copy_(w)
        assert all(torch.equal(a, b) for a, b in zip(df.quantize_experts(view), want)), off


@pytest.mark.parametrize("rows,E,K,N", [(3000, 1024, 16, 40), (3000, 64, 256, 1600), (40_000, 100, 64, 36), (9000, 30, 512, 1600)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_overlapping_offsets(dev, rows, E, K, N, dt):
    """Every other expert claims all rows: values mean nothing, but nothing outside the output is written, the call ends
    as soon as a right one would, and a right one after it is right."""
    g = torch.Generator(device=dev).manual_seed(rows)
    x, w = codes(g, dev, (rows, K), E4), codes(g, dev, (E, N, K), E4)
    s, sw = torch.ones(1, device=dev), torch.ones(E, device=dev)
    room = torch.full((rows + 600, N), 5.0, dtype=dt, device=dev)
    out = room[300:300 + rows]
    for bad in ([0, rows] * E, [rows, -3] * E, [0] + [rows] * E, [2 ** 31 - 1, -2 ** 31] * E):
        df.experts_fwd(x, w, torch.tensor(bad[:E + 1], dtype=torch.int64).to(torch.int32).to(dev), K, s, sw, out=out)
        assert (room[:300] == 5).all() and (room[300 + rows:] == 5).all()
    cut = torch.linspace(0, rows, E + 1, device=dev).int()
    df.experts_fwd(x, w, cut, K, s, sw, out=out)
    b = cut.tolist()
    ref = torch.cat([x[lo:hi].view(E4).float() @ w[e].view(E4).float().t() for e, (lo, hi) in enumerate(zip(b, b[1:]))])
    assert torch.equal(out, ref.to(dt))
