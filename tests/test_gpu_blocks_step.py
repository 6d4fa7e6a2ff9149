"""Runs of the calls with a scale per 128 values as a program makes them: a training
step through norm, quantizers and products with their gradients, a token's way through
norm, Linear and experts; eager, on another stream, and captured in a graph that is
replayed between the program's own eager work.

Gradients are checked against the formulas in binary64 on the codes as made (the
quantizers are tested by themselves): the products' bars are those of
test_gpu_blocks_gemm.py (2^-10 of the sum of magnitudes, half a step of the output),
the norm's those of test_gpu_rmsnorm.py.
"""
import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
U32 = torch.finfo(torch.float32).eps / 2


def values(q, s, K):
    return q[:, :K].double() * s.double().t().repeat_interleave(128, 1)[:, :K]


def near(got, a, b, bias=None):
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    u = torch.finfo(got.dtype).eps / 2
    assert ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -10 * size + 1e-30).all()


class Block:
    """norm(x + r) W^T + b, with its backward."""

    def __init__(self, dev, rows, K, N, scale_dtype, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        n = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.x, self.r, self.gamma = n(rows, K).to(BF), (n(rows, K) * 0.3).to(BF), (1 + 0.1 * n(K)).to(BF)
        self.w, self.b, self.dy = (n(N, K) * 0.02).to(BF), (n(N) * 0.1).to(BF), (n(rows, N) * 1e-3).to(BF)
        self.ds, self.kind, self.sizes = (n(rows, K) * 1e-2).to(BF), scale_dtype, (rows, K, N)

    def step(self):
        rows, K, N = self.sizes
        q = lambda t, **kw: df.quantize_blocks(t, want_qt=True, scale_dtype=self.kind, **kw)
        y, s, rstd = df.rmsnorm_forward(self.x, self.gamma, residual=self.r)
        xq, sx, xt, sxt = q(y)
        wq, sw, wt, swt = q(self.w, square=True)
        out = df.gemm_blocks(xq, sx, wq, sw, K, bias=self.b)
        dyq, sdy, dyt, sdyt = q(self.dy, fmt=df.Fmt.E5M2)
        dxn = df.gemm_blocks(dyq, sdy, wt, swt, N)
        dw = df.gemm_blocks(dyt, sdyt, xt, sxt, rows, out_dtype=torch.float32)
        dx, dg = df.rmsnorm_backward(dxn, s, self.gamma, rstd, dresidual=self.ds)
        return dict(y=y, s=s, rstd=rstd, xq=xq, sx=sx, xt=xt, sxt=sxt, wq=wq, sw=sw, wt=wt, swt=swt, out=out, dyq=dyq, sdy=sdy,
                    dyt=dyt, sdyt=sdyt, dxn=dxn, dw=dw, dx=dx, dg=dg)


def bits(t):
    return t.contiguous().view(torch.uint8)


def same(a, b):
    return all(torch.equal(bits(a[k]), bits(b[k])) for k in a)


@pytest.mark.parametrize("kind", [torch.float8_e8m0fnu, torch.float32])
@pytest.mark.parametrize("rows,K,N", [(200, 257, 130), (1000, 771, 520), (48, 1600, 640)])
def test_training_step(dev, kind, rows, K, N):
    blk = Block(dev, rows, K, N, kind)
    o = blk.step()
    assert torch.equal(o["s"], (blk.x.float() + blk.r.float()).to(BF))
    X, W = values(o["xq"], o["sx"], K), values(o["wq"], o["sw"], K)
    dY, dYt, Xt = values(o["dyq"], o["sdy"], N), values(o["dyt"], o["sdyt"], rows), values(o["xt"], o["sxt"], rows)
    assert torch.equal(values(o["wt"], o["swt"], N), W.t())  # squares: the same weights both ways
    near(o["out"], X, W, blk.b)
    near(o["dxn"], dY, W.t())
    near(o["dw"], dYt, Xt)
    # the norm's gradient on the dX that reached it
    s, rs = o["s"].double(), o["rstd"].double()[:, None]
    xh, g = s * rs, o["dxn"].double() * blk.gamma.double()
    m = (g * xh).mean(1, keepdim=True)
    want = rs * (g - xh * m) + blk.ds.double()
    size = rs * (g.abs() + xh.abs() * (g * xh).abs().mean(1, keepdim=True)) + blk.ds.double().abs()
    assert ((o["dx"].double() - want).abs() <= 2.0 ** -8 * want.abs() + 64 * U32 * size).all()
    t = o["dxn"].double() * xh
    assert ((o["dg"].double() - t.sum(0)).abs() <= (rows / 8 + 128) * U32 * t.abs().sum(0)).all()


@pytest.mark.parametrize("rows,K,N", [(200, 257, 130), (2048, 768, 2304)])
def test_training_step_on_another_stream_and_captured(dev, rows, K, N):
    blk, other = Block(dev, rows, K, N, torch.float8_e8m0fnu), Block(dev, rows, K, N, torch.float8_e8m0fnu, seed=1)
    want = [b.step() for b in (blk, other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = blk.step()
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = blk.step()
    inputs = [t.clone() for t in (blk.x, blk.r, blk.w, blk.dy, blk.gamma, blk.b, blk.ds)]
    for i in range(4):
        src = inputs if i % 2 == 0 else (other.x, other.r, other.w, other.dy, other.gamma, other.b, other.ds)
        for dst, t in zip((blk.x, blk.r, blk.w, blk.dy, blk.gamma, blk.b, blk.ds), src):
            dst.copy_(t)
        graph.replay()
        eager = blk.step()  # the program's own work between the replays
        torch.cuda.synchronize()
        assert same(captured, want[i % 2]) and same(eager, want[i % 2])


class Token:
    """What generating a token takes of these calls: norm, Linear, norm, experts."""

    def __init__(self, dev, tokens, H=320, N=192, experts=12, top=3, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        n = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.x, self.gamma, self.top = n(tokens, H).to(BF), (1 + 0.1 * n(H)).to(BF), top
        self.w = df.quantize_blocks(n(H, H) * H ** -0.5, square=True)[:2]
        self.router = df.quantize_blocks(n(experts, H) * H ** -0.5, square=True)[:2]
        self.w1 = df.quantize_experts_blocks(n(experts, 2 * N, H) * H ** -0.5)
        self.w2 = df.quantize_experts_blocks(n(experts, H, N) * N ** -0.5)
        self.H = H

    def step(self):
        q, sq, _, _ = df.rmsnorm_quantize(self.x, self.gamma)
        h = df.gemm_blocks(q, sq, *self.w, self.H)
        q2, sq2, s, _, y = df.rmsnorm_quantize(h, self.gamma, residual=self.x, want_y=True)
        logits = df.gemm_blocks(q2, sq2, *self.router, self.H, out_dtype=torch.float32)
        out, ids, wt = df.moe_layer(y, logits, *self.w1, *self.w2, self.top)
        return dict(h=h, s=s, y=y, logits=logits, out=out, ids=ids, wt=wt)


@pytest.mark.parametrize("tokens", [1, 2, 40])
def test_token_captured(dev, tokens):
    """Two graphs, and eager work between their replays: each keeps its own workspace."""
    tok = [Token(dev, tokens, seed=i) for i in range(2)]
    want = [t.step() for t in tok]
    graphs, captured = [], []
    for t in tok:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            captured.append(t.step())
    for i in (0, 1, 1, 0, 0):
        for v in captured[i].values():
            v.fill_(1)
        graphs[i].replay()
        eager = tok[1 - i].step()
        torch.cuda.synchronize()
        assert same(captured[i], want[i]) and same(eager, want[1 - i])


def test_two_layers_at_once(dev):
    """Two streams run the experts' layer at the same time."""
    tok = [Token(dev, 48, H=1024, N=512, seed=i) for i in range(2)]
    want = [t.step() for t in tok]
    streams = [torch.cuda.Stream() for _ in tok]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tok[i].step())
    torch.cuda.synchronize()
    assert all(same(g, want[i]) for i in range(2) for g in got[i])


# sizes on both sides of the choice of kernel, odd ones: 16 x 16, 16 x 32, 32 x 32 (four and
# eight waves), 64 x 64, 128 x 128, 256 x 128, 256 x 256
KERNELS = [(16, 33, 300), (9, 5003, 1100), (70, 1601, 300), (70, 6403, 1601), (260, 6401, 1601), (1030, 1603, 1601),
           (300, 6200, 1600), (4100, 1603, 1599), (2050, 6403, 1601), (1027, 1601, 4001)]


@pytest.mark.parametrize("kind", [torch.float8_e8m0fnu, torch.float32])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", KERNELS)
def test_every_kernel(dev, kind, out, M, N, K):
    g = torch.Generator(device=dev).manual_seed(M)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)
    a = n(M, K) * torch.exp(2 * n(M, 1))
    w = n(N, K) * 0.02
    bias = n(N).to(BF)
    for square, fmt in ((True, df.Fmt.E4M3), (False, df.Fmt.E5M2)):
        aq, sa, _, _ = df.quantize_blocks(a, fmt, scale_dtype=kind)
        bq, sb, _, _ = df.quantize_blocks(w, square=square, scale_dtype=kind)
        got = df.gemm_blocks(aq, sa, bq, sb, K, bias=bias if square else None, out_dtype=out)
        va, vb = values(aq, sa, K), values(bq, sb, K)
        want, size = va @ vb.t(), va.abs() @ vb.abs().t()
        if square:
            want, size = want + bias.double(), size + bias.double().abs()
        u = torch.finfo(out).eps / 2
        bar = (K + 64) * U32 * size if out == torch.float32 else u * want.abs() + 2.0 ** -10 * size + 6e-8
        assert ((got.double() - want).abs() <= bar).all()
