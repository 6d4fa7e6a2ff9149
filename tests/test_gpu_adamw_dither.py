"""df_adamw_update_dithered: bit for bit against its rule in numpy, and over
thousands of steps against 32-bit states.

The bars of the long runs.  A kept root is drawn so that its mean is right; a
move of a share d of a code gap w (relative, at most 1/8) is made with probability
d and adds a relative variance of d w^2.  While gradients stay as they are d w is
at most (1 - b2) (half of it the root's own move, half the scale's) and b2^2 of a
variance is left after each further step: 1 / (8 (1 + b2)) in all, at most 0.0642
from b2 = 0.95 up, a standard deviation below 0.26.  While roots fall, nothing
draws them back: their moves add up to the fall's logarithm, ln 10 = 2.31, and the
variances to 2.31 / 8 more, 0.36 in all.  The next root is a convex function of
the kept one (that of b2 r^2 plus the gradient's part), which takes the mean up by
half the relative variance at most.  So over N independent values the mean of kept
root over true root lies within half the variance and 6 deviations / sqrt(N) of 1,
and its variance is below the one above.
"""
import numpy as np
import pytest
import torch

import deepfuse_amd as df
from test_gpu_adamw import F, HYPER, SIZES, blocks, dev_list, host, make, same, scales, step32, widen

pytestmark = pytest.mark.gpu

U = np.uint32


def mix(x):
    x = np.array(x, dtype=U)
    with np.errstate(over="ignore"):
        x ^= x >> U(16)
        x *= U(0x6A09E667)
        x ^= x >> U(15)
        x *= U(0xBB67AE85)
    return x ^ (x >> U(16))


def draws(seed, t, idx, i):
    i = np.asarray(i, dtype=np.uint64)
    with np.errstate(over="ignore"):
        key = mix(mix(mix(U(seed)) + U(t)) + U(idx))
        return mix(key + (i & np.uint64(0xFFFFFFFF)).astype(U) * U(0x9E3779B9) + (i >> np.uint64(32)).astype(U) * U(0xBB67AE85))


def dither(q, r):
    """e4m3 codes of binary32 q by 16 random bits each"""
    a = np.abs(q)
    with np.errstate(all="ignore"):
        up = np.where(a < F(2.0 ** -6), F(2.0 ** -6), F(0))  # below it the steps are those above it
        n = (((a + up).view(U) + (r << U(4)) + U(8)) & U(0xFFF00000)).view(F) - up
        z = np.copysign(np.minimum(n, F(448)), q).astype(F)
        z = np.where(a <= F(448), z, np.clip(q, F(-448), F(448)))
    c = torch.from_numpy(z).to(torch.float8_e4m3fn)
    back = c.float().numpy()
    assert np.array_equal(back[np.isfinite(z)], z[np.isfinite(z)])  # an e4m3 value each
    return c.view(torch.uint8).numpy()


def keep(x, rnd, root=False):
    with np.errstate(all="ignore"):
        y = np.sqrt(x) if root else x
        s = scales(y)
        q = (blocks(y) * (F(1) / s)[:, None]).reshape(-1)[:len(x)].astype(F)
    if root:
        q = np.where(y > 0, np.maximum(q, F(2.0 ** -9)), q).astype(F)
    return dither(q, (rnd >> U(16)) if root else (rnd & U(0xFFFF))), s


def check_steps(dev, p, g, gdt, steps, seed, copy=None, wd=0.1, beta2=0.95):
    P, G = dev_list(p, dev), [t.to(dev) for t in g]
    M, V, MS, VS = df.adamw_state(P, 8)
    copies = None if copy is None else [torch.zeros_like(t, dtype=copy) for t in P]
    m, v = [np.zeros_like(a) for a in p], [np.zeros_like(a) for a in p]
    for t in steps:
        df.adamw_update(P, G, M, V, t, lr=3e-3, beta1=0.9, beta2=beta2, eps=1e-8, weight_decay=wd, m_scales=MS, v_scales=VS,
                        copies=copies, dither=seed)
        for i in range(len(p)):
            p[i], m[i], v[i] = step32(p[i], g[i].float().numpy(), m[i], v[i], t, wd, beta2=beta2)
            r = draws(seed & 0xFFFFFFFF, t, i, np.arange(len(p[i])))
            (cm, sm), (cv, sv) = keep(m[i], r), keep(v[i], r, root=True)
            assert same(host(P)[i], p[i]) and same(host(MS)[i], sm) and same(host(VS)[i], sv), (t, i)
            nan = lambda c: (c & 0x7F) == 0x7F
            for got, want in ((host(M)[i], cm), (host(V)[i], cv)):
                assert np.array_equal(nan(got), nan(want)) and same(got[~nan(want)], want[~nan(want)]), (t, i)
            if copy is not None:
                assert torch.equal(copies[i].cpu(), torch.from_numpy(p[i]).to(copy)), (t, i)
            m[i], v[i] = widen(host(MS)[i], host(M)[i]), widen(host(VS)[i], host(V)[i], root=True)


@pytest.mark.parametrize("gdt,copy", [(torch.float32, None), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                      (torch.bfloat16, None), (torch.float32, torch.float16)])
@pytest.mark.parametrize("seed", [0, 12345, -1])
def test_steps_bit_exact(dev, gdt, copy, seed):
    p, g = make(SIZES, 5, gdt)
    check_steps(dev, p, g, gdt, (1, 2, 3, 100, 101), seed, copy)


def test_long_list(dev):
    """More tensors than a launch holds: each draws by its place in the caller's list, empty ones counted."""
    p, g = make([(i * 37) % 700 for i in range(95)], 6, torch.float32)
    check_steps(dev, p, g, torch.float32, (1, 2), 7)


@pytest.mark.parametrize("beta2", [0.95, 0.999])
def test_magnitudes_and_not_finite(dev, beta2):
    """Units of values of each size, zeros of both signs, infinities and NaN, roots far below their block's largest."""
    rng = np.random.default_rng(11)
    n = 256 * 4 * 40
    g = (rng.standard_normal(n) * np.repeat(np.exp2(np.linspace(-149, 40, n // 256)), 256)).astype(F)
    g[rng.random(n) < 0.05] = 0.0
    g[rng.random(n) < 0.05] = -0.0
    g[5000:5256] = np.logspace(-30, 0, 256)
    g[9000] = np.inf
    g[9300] = -np.inf
    g[9600] = np.nan
    for tail in (0, 13):
        p = [(rng.standard_normal(n + tail) * 0.1).astype(F)]
        check_steps(dev, p, [torch.from_numpy(np.concatenate([g, g[:tail]]))], torch.float32, (1, 2, 3), 3, beta2=beta2)


def test_no_step_but_codes(dev):
    """Parameters, scales and absmax are those of the undithered step; a code moves to a neighbour at most."""
    p, g = make([70_001], 8, torch.float32)
    runs = []
    for d in (None, 9):
        P, G = dev_list(p, dev), [t.to(dev) for t in g]
        M, V, MS, VS = df.adamw_state(P, 8)
        am = torch.zeros(1, device=dev)
        df.adamw_update(P, G, M, V, 1, m_scales=MS, v_scales=VS, absmax=am, dither=d)
        runs.append([P[0], MS[0], VS[0], am, M[0].view(torch.uint8), V[0].view(torch.uint8)])
    for a, b in zip(runs[0][:4], runs[1][:4]):
        assert torch.equal(a, b)
    for a, b in zip(runs[0][4:], runs[1][4:]):
        d = ((a & 0x7F).int() - (b & 0x7F).int()).abs()
        assert d.max() == 1 and 0.1 < d.float().mean() < 0.4  # a nearest code is left with half the distance's share: 1/4


@pytest.mark.parametrize("beta2,before,after", [(0.95, 200, 400), (0.99, 600, 1500), (0.999, 3000, 8000)])
@pytest.mark.parametrize("noisy", [False, True])
def test_v_follows_a_fall(dev, beta2, before, after, noisy):
    """Half of each block's gradients fall tenfold: the kept v follows the one in 32 bits, at every b2."""
    n = 64 * 256
    size = torch.ones(64, 256, device=dev)
    G = torch.Generator(device=dev).manual_seed(4)
    p8, p32, g = [torch.zeros(n, device=dev)], [torch.zeros(n, device=dev)], [torch.ones(n, device=dev)]
    s8, s32 = df.adamw_state(p8, 8), df.adamw_state(p32)
    at = {before + int(k / (1 - beta2)) for k in (0, 0.5, 2, 5)} | {before + after}
    for t in range(1, before + after + 1):
        if t == before + 1:
            size[:, 128:] = 0.1
        if noisy:
            torch.randn(64, 256, generator=G, device=dev, out=g[0].view(64, 256))
            g[0].view(64, 256).mul_(size)
        else:
            g[0].view(64, 256).copy_(size)
        df.adamw_update(p8, g, s8[0], s8[1], t, beta2=beta2, m_scales=s8[2], v_scales=s8[3], dither=1)
        df.adamw_update(p32, g, s32[0], s32[1], t, beta2=beta2)
        if t in at:
            r = (s8[1][0].float().view(-1, 256) * s8[3][0][:, None]).double() / s32[1][0].double().sqrt().view(-1, 256)
            for x, var in ((r[:, :128], 0.0642), (r[:, 128:], 0.36)):
                assert abs(x.mean().item() - 1) <= var / 2 + 6 * (var / x.numel()) ** 0.5, (t, x.mean().item())
                assert x.var().item() <= var, t


def test_moments_vanish_together(dev):
    """Gradients that end: m falls by b1 and sqrt(v) by the root of b2 a step, so the steps end too, and do not grow."""
    n = 64 * 256
    p, g = [torch.zeros(n, device=dev)], [torch.ones(n, device=dev)]
    st = df.adamw_state(p, 8)
    step = lambda t: df.adamw_update(p, g, st[0], st[1], t, lr=1.0, beta1=0.95, beta2=0.99, weight_decay=0.0, m_scales=st[2],
                                     v_scales=st[3], dither=2)
    for t in range(1, 101):
        step(t)
    g[0].view(64, 256)[:, 1:] = 0  # one value keeps its gradient, and the block its scale
    for t in range(101, 161):
        step(t)
    m = (st[0][0].float().view(-1, 256) * st[2][0][:, None])[:, 1:]
    # 0.95^60 = 0.046.  Nothing draws a value back here: relative variances of 0.05 / 8 a step (move 0.05, gap 1/8) add up
    # over 60 steps to e^0.375 - 1 = 0.45, a deviation of 0.67 / sqrt(16320) = 0.005 of the mean
    assert abs(m.mean().item() / 0.95 ** 60 / (1 - 0.95 ** 100) - 1) <= 0.05
    before = p[0].clone()
    for t in range(161, 200):
        step(t)
    moved = (p[0] - before).view(64, 256)[:, 1:].abs().mean().item()
    # in 32 bits: sum over k of 0.95^k / 0.995^k from k = 61 to 99, bias corrections 1 - 0.95^t and 1 - 0.99^t (0.8 to 0.87)
    want = sum((0.95 ** k / (1 - 0.95 ** (100 + k))) / (0.99 ** (k / 2) * ((1 - 0.99 ** 100) / (1 - 0.99 ** (100 + k))) ** 0.5)
               for k in range(61, 100)) * (1 - 0.95 ** 100)
    # the mean of 1 / root lies above 1 / its mean by about the relative variance, 0.005 / 8 a step over 60 to 100 steps
    # (0.04 to 0.06); m's mean is off by e^0.62 - 1 = 0.86 at most, 0.93 / sqrt(16320) = 0.007 of it
    assert 0.95 * want <= moved <= 1.15 * want


def test_captured_steps_draw_anew(dev):
    """The draw follows the device's step count on replay, and equals the eager call's; another seed, other codes."""
    p, g = make([5000, 257], 9, torch.bfloat16)
    P, G = dev_list(p, dev), [t.to(dev) for t in g]
    Q = [t.clone() for t in P]
    a, b = df.adamw_state(P, 8), df.adamw_state(Q, 8)
    step = torch.zeros(1, dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        df.adamw_update(P, G, a[0], a[1], step, m_scales=a[2], v_scales=a[3], dither=5)
    for t in range(1, 6):
        graph.replay()
        df.adamw_update(Q, G, b[0], b[1], t, m_scales=b[2], v_scales=b[3], dither=5)
        torch.cuda.synchronize()
        for x, y in zip((P, *a), (Q, *b)):
            assert all(torch.equal(u.view(torch.uint8), w.view(torch.uint8)) for u, w in zip(x, y)), t
    codes = []
    for seed in (5, 6):
        c = [[t.clone() for t in x] for x in (Q, *b)]
        df.adamw_update(c[0], G, c[1], c[2], 6, m_scales=c[3], v_scales=c[4], dither=seed)
        codes.append(c[2][0].view(torch.uint8))
    assert not torch.equal(*codes)


def test_views_and_large_lists(dev):
    """Odd elements, and a list past 256 MB: the same codes."""
    n, big = 8192 * 2 + 1300, 40_000_000
    p, g = make([n], 13, torch.bfloat16)
    runs = []
    for k, extra in ((0, 0), (1, 0), (3, big)):
        at = lambda t: torch.cat([torch.zeros(k * t.element_size(), dtype=torch.uint8, device=dev), t.view(torch.uint8).reshape(-1),
                                  torch.zeros(16, dtype=torch.uint8, device=dev)]
                                 )[k * t.element_size():][:t.numel() * t.element_size()].view(t.dtype)
        P, G = [at(t) for t in dev_list(p, dev)], [at(t.to(dev)) for t in g]
        st = [[at(x[0])] for x in df.adamw_state(P, 8)]
        if extra:
            P.append(torch.ones(extra, device=dev))
            G.append(torch.zeros(extra, dtype=torch.bfloat16, device=dev))
            st = [x + y for x, y in zip(st, df.adamw_state(P[1:], 8))]
        for t in (1, 2):
            df.adamw_update(P, G, st[0], st[1], t, m_scales=st[2], v_scales=st[3], dither=0, **HYPER)
        runs.append([x[0].clone() for x in (P, *st)])
    for other in runs[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(runs[0], other))
