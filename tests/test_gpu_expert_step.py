"""A training step of a norm in front of a Linear dealt to experts, as it is
used: residual add and LayerNorm, fp8 codes, the experts' products, their
gradients, the norm's gradient, clipping's norm and the AdamW update with 8-bit
states, every part of it next to binary64 on what the part before gave; then the
same step captured in a graph and replayed over changing inputs, routing, step
count and rate, equal bit for bit to the eager step.
"""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import Fmt

pytestmark = pytest.mark.gpu

T, D, H, E = 700, 400, 272, 6
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


class Model:
    def __init__(self, dev, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        r = lambda *s, std=1.0: torch.randn(*s, generator=g, device=dev) * std
        self.params = [1 + r(D, std=0.1), r(D, std=0.1), r(E, H, D, std=0.05)]  # gamma, beta, w
        self.copies = [p.bfloat16() for p in self.params]
        self.state = df.adamw_state(self.params, 8)
        self.x, self.res, self.dy = (r(T, D).bfloat16(), r(T, D, std=0.5).bfloat16(), r(T, H, std=1e-2).bfloat16())
        self.dres = r(T, D, std=1e-2).bfloat16()
        self.off = torch.zeros(E + 1, dtype=torch.int32, device=dev)
        self.step = torch.zeros(1, dtype=torch.int32, device=dev)
        self.lr = torch.full((1,), 1e-3, device=dev)
        self.am = torch.zeros(3, device=dev)
        # rows behind the last expert keep what these hold
        self.y, self.dh = torch.zeros(T, H, dtype=torch.bfloat16, device=dev), torch.zeros(T, D, dtype=torch.bfloat16, device=dev)

    def route(self, counts):
        self.off.copy_(torch.tensor([0] + counts, dtype=torch.int32).cumsum(0, dtype=torch.int32))

    def run(self):
        """one step; what it computed, by name"""
        gamma, beta, w = self.copies
        h, s, mean, rstd = df.layernorm_forward(self.x, gamma, beta, residual=self.res)
        _, sh, hq, hqt = df.quantize_2d_jit(h, Fmt.E4M3, want_qt=True)
        sw, wq, wqt = df.quantize_experts(w)
        y = df.experts_fwd(hq, wq, self.off, D, sh, sw, out=self.y)
        _, sdy, dyq, dyqt = df.quantize_2d_jit(self.dy, Fmt.E5M2, want_qt=True)
        dh = df.experts_dx(dyq, wqt, self.off, H, sdy, sw, out=self.dh)
        dw = df.experts_dw(dyqt, hqt, self.off, T, sdy, sh)
        dx, dgamma, dbeta = df.layernorm_backward(dh, s, gamma, mean, rstd, dresidual=self.dres)
        grads = [dgamma, dbeta, dw]
        norm = df.grad_norm(grads)
        self.step.add_(1)
        df.adamw_update(self.params, grads, self.state[0], self.state[1], self.step, lr=self.lr, weight_decay=[0.0, 0.0, 0.1],
                        m_scales=self.state[2], v_scales=self.state[3], copies=self.copies, clip_norm=norm, max_norm=0.5,
                        absmax=self.am)
        return dict(h=h, s=s, hq=hq, sh=sh, wq=wq, sw=sw, y=y, dyq=dyq, sdy=sdy, dh=dh, dw=dw, dx=dx, dgamma=dgamma, dbeta=dbeta,
                    norm=norm, mean=mean, rstd=rstd)

    def everything(self):
        return [*self.params, *self.copies, *[t.view(torch.uint8) for t in self.state[0] + self.state[1]], *self.state[2],
                *self.state[3], self.y, self.dh, self.am]


def near(got, want, size, n):
    """one rounding to the type of a binary32 sum of n terms of total size `size`; from fp8 products (2-byte outputs) 7 * 2^-13
    of it as well"""
    rel = 2 * (n + 70) * 2.0 ** -24 + (0 if got.dtype == torch.float32 else 7 * 2.0 ** -13)
    assert ((got.double() - want).abs() <= U[got.dtype] * want.abs() + rel * size + 1e-30).all()


@pytest.mark.parametrize("counts", [[100, 0, 250, 1, 149, 200], [30, 10, 0, 500, 20, 40]])
def test_parts_against_binary64(dev, counts):
    m = Model(dev)
    m.route(counts)
    before = [p.clone() for p in m.params]
    gamma = m.copies[0].double()  # the step writes the copies
    o = {k: v.clone() for k, v in m.run().items()}
    b = m.off.tolist()
    used = b[-1]
    hd, dyd = o["hq"].view(E4)[:, :D].double() * o["sh"].double(), o["dyq"].view(E5)[:, :H].double() * o["sdy"].double()
    wd = o["wq"].view(E4)[..., :D].double() * o["sw"].double()[:, None, None]
    # the codes stand for what was quantized: half a step of e4m3 (2^-4 of the value, 2^-10 of the scale)
    assert ((hd - o["h"].double()).abs() <= 2.0 ** -4 * o["h"].double().abs() + 2.0 ** -9 * o["sh"].double()).all()
    for e, (lo, hi) in enumerate(zip(b, b[1:])):
        near(o["y"][lo:hi], hd[lo:hi] @ wd[e].t(), hd[lo:hi].abs() @ wd[e].abs().t(), D)
        near(o["dh"][lo:hi], dyd[lo:hi] @ wd[e], dyd[lo:hi].abs() @ wd[e].abs(), H)
        near(o["dw"][e], dyd[lo:hi].t() @ hd[lo:hi], dyd[lo:hi].abs().t() @ hd[lo:hi].abs(), hi - lo)
    assert not o["y"][used:].any() and not o["dh"][used:].any()
    # the norm's gradient by autograd in binary64
    s = o["s"].double().requires_grad_()
    ga = gamma.clone().requires_grad_()
    be = torch.zeros(D, dtype=torch.float64, device=dev, requires_grad=True)
    torch.nn.functional.layer_norm(s, (D,), ga, be, 1e-5).backward(o["dh"].double())
    for got, want in ((o["dx"], s.grad + m.dres.double()), (o["dgamma"], ga.grad), (o["dbeta"], be.grad)):
        size = want.abs().mean() * 30  # sums of 400 to 700 terms that partly cancel
        assert ((got.double() - want).abs() <= U[got.dtype] * want.abs() + 1000 * 2.0 ** -24 * size).all()
    total = sum((o[k].double() ** 2).sum() for k in ("dgamma", "dbeta", "dw")).sqrt()
    assert abs(o["norm"].double() - total) <= 2.0 ** -22 * total
    # the first step moves a parameter by at most lr (m / sqrt(v) is 1 there) and its decay
    for p, q, wd_ in zip(m.params, before, (0, 0, 0.1)):
        assert ((p - q).abs() <= 1.001e-3 + 1.001e-3 * wd_ * q.abs()).all()
    assert all(torch.equal(c, p.bfloat16()) for c, p in zip(m.copies, m.params))
    assert all(am == p.abs().max() for am, p in zip(m.am, m.params))


def test_captured_step(dev):
    eager, captured = Model(dev), Model(dev)
    captured.route([10] * E)
    captured.run()  # before capture: nothing is left to be set up
    captured = Model(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.run()
    assert captured.step.item() == 0
    for k, counts in enumerate(([100, 0, 250, 1, 149, 200], [700, 0, 0, 0, 0, 0], [1, 2, 3, 4, 5, 6], [0] * 6,
                                [116, 117, 116, 117, 117, 117])):
        for m in (eager, captured):
            m.route(counts)
            m.lr.fill_(1e-3 * (k + 1))
            m.x.copy_(torch.randn(T, D, generator=torch.Generator(device=dev).manual_seed(k), device=dev))
        eager.run()
        graph.replay()
        torch.cuda.synchronize()
        assert captured.step.item() == k + 1
        for i, (a, b) in enumerate(zip(eager.everything(), captured.everything())):
            assert torch.equal(a, b), (k, i)


def test_gradient_against_differences(dev):
    """The step's dW against differences of sum(dy * y) in the experts' weights (binary64, on the codes' values)."""
    m = Model(dev)
    counts = [100, 0, 250, 1, 149, 200]
    m.route(counts)
    o = m.run()
    b = m.off.tolist()
    hd, dyd = o["hq"].view(E4)[:, :D].double() * o["sh"].double(), o["dyq"].view(E5)[:, :H].double() * o["sdy"].double()
    f = lambda w: sum((dyd[lo:hi] * (hd[lo:hi] @ w[e].t())).sum() for e, (lo, hi) in enumerate(zip(b, b[1:])))
    g = torch.Generator(device=dev).manual_seed(3)
    d = torch.randn(E, H, D, generator=g, device=dev, dtype=torch.float64)
    w = o["wq"].view(E4)[..., :D].double() * o["sw"].double()[:, None, None]
    num = (f(w + d) - f(w - d)) / 2  # f is linear in w
    got = (o["dw"].double() * d).sum()
    assert abs(got - num) <= 2.0 ** -20 * (o["dw"].double() * d).abs().sum()
