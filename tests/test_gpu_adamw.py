"""df_adamw_update and df_grad_norm: bit for bit against the same operations,
each rounded to binary32, in numpy, and within derived bars of the formula in
binary64; lists ragged around the 256 values of a scale, the 1024 whose loads
are in flight together, the 8192 of a block, and longer than a launch holds (40).
"""
import numpy as np
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import DType

pytestmark = pytest.mark.gpu

F = np.float32
SIZES = [0, 1, 3, 255, 256, 257, 1023, 1024, 1025, 8191, 8192, 8193, 3 * 8192 + 1285, 100_003]
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8)


def bias_corr(beta, t):
    return F(1) - F(np.float64(F(beta)) ** t)


def e4m3(x):
    """codes of binary32 x (saturating, NaN as 0x7F with its sign)"""
    t = torch.from_numpy(np.clip(x, F(-448), F(448)))
    return t.to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def decode(c):
    return torch.from_numpy(c).view(torch.float8_e4m3fn).float().numpy()


def blocks(x):
    return np.pad(x, (0, -len(x) % 256)).reshape(-1, 256)


def scales(x):
    a = np.abs(blocks(x))
    big = np.where(np.isfinite(a), a, 0).max(1)
    return np.where(big > 0, np.maximum(big / F(448), F(2.0 ** -126)), F(1)).astype(F)


def step32(p, g, m, v, t, wd, f=F(1), lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8):
    """one step of one tensor in binary32: new p, m, v"""
    lr, b1, b2, eps, wd = F(lr), F(beta1), F(beta2), F(eps), F(wd)
    with np.errstate(all="ignore"):
        g = g.astype(F) * f
        m = b1 * m + (F(1) - b1) * g
        v = b2 * v + (F(1) - b2) * g * g
        p = p * (F(1) - lr * wd) - lr * (m / bias_corr(b1, t)) / (np.sqrt(v / bias_corr(b2, t)) + eps)
    return p, m, v


def widen(s, c, root=False):
    x = (blocks(decode(c)) * s[:, None]).reshape(-1)[:len(c)]
    return x * x if root else x


def keep8(x, root=False):
    """codes and scales of a new state"""
    with np.errstate(all="ignore"):
        y = np.sqrt(x) if root else x
        s = scales(y)
        q = (blocks(y) / s[:, None]).reshape(-1)[:len(x)]
    if root:
        q = np.where(y > 0, np.maximum(q, F(2.0 ** -9)), q).astype(F)
    return e4m3(q), s


def same(a, b):
    """equal bits, any NaN for any NaN"""
    a, b = np.asarray(a), np.asarray(b)
    if a.dtype == np.uint8:
        return np.array_equal(a, b)
    both = np.isnan(a) & np.isnan(b)
    return np.array_equal(np.where(both, 0, a.view(np.int32)), np.where(both, 0, b.view(np.int32)))


def make(sizes, seed, gdt, std=1e-3):
    rng = np.random.default_rng(seed)
    p = [(rng.standard_normal(n) * 0.02).astype(F) for n in sizes]
    g = [torch.from_numpy((rng.standard_normal(n) * std * np.exp(2 * rng.standard_normal())).astype(F)).to(gdt) for n in sizes]
    return p, g


def dev_list(arrays, dev):
    return [torch.from_numpy(np.array(a)).to(dev) for a in arrays]


def host(ts):
    return [(t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).cpu().numpy() for t in ts]


@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("copy", [None, torch.bfloat16, torch.float16])
def test_steps_bit_exact(dev, gdt, bits, copy):
    p, g = make(SIZES, 5, gdt)
    P, G = dev_list(p, dev), [t.to(dev) for t in g]
    M, V, MS, VS = df.adamw_state(P, bits)
    copies = None if copy is None else [torch.zeros_like(t, dtype=copy) for t in P]
    am = torch.full((len(P),), -1.0, device=dev)
    wd = [0.1 if i % 2 else 0.0 for i in range(len(P))]
    m, v = [np.zeros_like(a) for a in p], [np.zeros_like(a) for a in p]
    for t in (1, 2, 3):
        df.adamw_update(P, G, M, V, t, weight_decay=wd, m_scales=MS, v_scales=VS, copies=copies, absmax=am, **HYPER)
        torch.cuda.synchronize()
        for i, n in enumerate(SIZES):
            p[i], m[i], v[i] = step32(p[i], g[i].float().numpy(), m[i], v[i], t, wd[i])
            assert same(host(P)[i], p[i]), (t, n)
            if bits == 32:
                assert same(host(M)[i], m[i]) and same(host(V)[i], v[i]), (t, n)
            else:
                (cm, sm), (cv, sv) = keep8(m[i]), keep8(v[i], root=True)
                assert same(host(M)[i], cm) and same(host(V)[i], cv), (t, n)
                assert same(host(MS)[i], sm) and same(host(VS)[i], sv), (t, n)
                m[i], v[i] = widen(sm, cm), widen(sv, cv, root=True)
            if copies is not None:
                assert torch.equal(copies[i].cpu(), torch.from_numpy(p[i]).to(copy)), (t, n)
            assert am[i].item() == (np.abs(p[i]).max() if n else 0.0)


def test_long_list_and_decay(dev):
    sizes = [(i * 37) % 700 for i in range(95)]
    p, g = make(sizes, 6, torch.float32)
    P, G = dev_list(p, dev), [t.to(dev) for t in g]
    M, V, _, _ = df.adamw_state(P)
    wd = [0.01 * (i % 5) for i in range(95)]
    df.adamw_update(P, G, M, V, 1, weight_decay=wd, **HYPER)
    for i in range(95):
        assert same(host(P)[i], step32(p[i], g[i].numpy(), 0 * p[i], 0 * p[i], 1, wd[i])[0]), i


@pytest.mark.parametrize("bits", [32, 8])
def test_against_binary64(dev, bits):
    """The formula in binary64 from the same state: p's error is the rounding of p*keep, of the step and of their
    difference (u each of their size), and the step's own: 12 roundings and what cancels in m."""
    p, g = make([50_000], 7, torch.float32)
    P, G = dev_list(p, dev), [t.to(dev) for t in g]
    M, V, MS, VS = df.adamw_state(P, bits)
    for t in range(1, 6):
        before = [x.double() for x in (P[0], G[0])]
        md, vd = (x[0].float().clone() for x in (M, V))  # the step writes them
        if bits == 8:
            pad = lambda x, s: (torch.nn.functional.pad(x, (0, -len(x) % 256)).view(-1, 256) * s[0][:, None]).view(-1)[:len(x)]
            md, vd = pad(md, MS), pad(vd, VS).square()
        df.adamw_update(P, G, M, V, t, weight_decay=0.1, m_scales=MS, v_scales=VS, **HYPER)
        b1, b2, lr, eps, wd = (float(F(x)) for x in (0.9, 0.95, 3e-3, 1e-8, 0.1))
        m1, m2 = b1 * md.double(), (1 - b1) * before[1]
        m, v = m1 + m2, b2 * vd.double() + (1 - b2) * before[1] ** 2
        scale = lr / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + eps)
        want = before[0] * (1 - lr * wd) - scale * m
        u = 2.0 ** -24
        # 1 - beta and 1 - beta^t are rounded constants: up to u / (1 - beta) of their value
        bar = 3 * u * before[0].abs() + (16 + 2 / (1 - b1) + 2 / (1 - b2)) * u * scale * (m1.abs() + m2.abs()) + u * want.abs()
        assert ((P[0].double() - want).abs() <= bar).all()
        if bits == 8:
            # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below its normal range), or code 1 for v
            for c, s, x, low in ((M, MS, m, 2.0 ** -10), (V, VS, v.sqrt(), 2.0 ** -9)):
                s = s[0].double().repeat_interleave(256)[:len(x)]
                got = c[0].double() * s
                assert ((got - x).abs() <= (2.0 ** -4 + 1e-6) * x.abs() + low * s).all()


def test_eight_bit_corners(dev):
    """Blocks of zeros, of one value, with infinities and NaN, of the smallest magnitudes; v far below its block's largest."""
    n = 256 * 8
    g = np.zeros(n, F)
    g[256:512] = 1e-3
    g[512:768] = np.logspace(-30, 0, 256)
    g[768] = np.inf
    g[769] = np.nan
    g[770:1024] = 0.5
    g[1024:1280] = 1e-38
    g[1280:1536] = 1e-45
    g[1536] = 3e38
    p = np.ones(n, F)
    P, G = dev_list([p], dev), dev_list([g], dev)
    M, V, MS, VS = df.adamw_state(P, 8)
    m = v = np.zeros(n, F)
    for t in (1, 2):
        am = torch.zeros(1, device=dev)
        df.adamw_update(P, G, M, V, t, weight_decay=0.0, m_scales=MS, v_scales=VS, absmax=am, **HYPER)
        p, m, v = step32(p, g, m, v, t, 0.0)
        (cm, sm), (cv, sv) = keep8(m), keep8(v, root=True)
        assert same(host(P)[0], p) and same(host(MS)[0], sm) and same(host(VS)[0], sv)
        finite = np.isfinite(m) & np.isfinite(v)
        assert same(host(M)[0][finite], cm[finite]) and same(host(V)[0][finite], cv[finite])
        assert ((host(M)[0][~np.isfinite(m)] & 0x7F) >= 0x7E).all()  # infinity saturated, NaN kept
        assert (host(V)[0][(v > 0) & np.isfinite(v)] > 0).all()  # never code 0
        assert am.item() == np.abs(p[np.isfinite(p)]).max()
        m, v = widen(host(MS)[0], host(M)[0]), widen(host(VS)[0], host(V)[0], root=True)
    assert np.isfinite(host(P)[0][512:768]).all()


@pytest.mark.parametrize("gdt", [torch.bfloat16, torch.float16, torch.float32])
def test_clip_from_the_norm(dev, gdt):
    sizes = [0, 5, 8192, 32768, 32769, 70_001]
    p, g = make(sizes, 8, gdt, std=1.0)
    P, G = dev_list(p, dev), [t.to(dev) for t in g]
    norm = df.grad_norm(G)
    want = np.sqrt(sum((t.double() ** 2).sum().item() for t in g))
    # squares rounded to binary32 (exact for 2-byte types), a binary64 sum, one rounding of the root
    assert abs(norm.item() - want) <= 2.0 ** -23 * want
    M, V, _, _ = df.adamw_state(P)
    df.adamw_update(P, G, M, V, 1, weight_decay=0.1, clip_norm=norm, max_norm=1.5, **HYPER)
    f = F(1.5) / F(norm.item())
    for i in range(len(sizes)):
        assert same(host(P)[i], step32(p[i], g[i].float().numpy(), 0 * p[i], 0 * p[i], 1, 0.1, f)[0])


@pytest.mark.parametrize("gdt", [torch.bfloat16, torch.float16])
def test_norm_of_unaligned_and_empty(dev, gdt):
    x = torch.randn(40_001, device=dev).to(gdt)
    cut = [x[1:40_000], x[3:3], x[40_000:]]
    want = np.sqrt(sum((t.double() ** 2).sum().item() for t in cut))
    assert abs(df.grad_norm(cut).item() - want) <= 2.0 ** -23 * want
    assert df.grad_norm([x[:0]]).item() == 0.0


@pytest.mark.parametrize("bits", [32, 8])
def test_views_at_any_element(dev, bits):
    """Parameters and states as views at odd offsets of larger buffers; what lies around them stays."""
    n, off = 5003, 1
    base = {k: torch.randn(n + 9, device=dev) for k in ("p", "g")}
    whole = [base["p"][off:off + n].clone()], [base["g"][off:off + n].clone()]
    st = df.adamw_state(whole[0], bits)
    views = [base["p"][off:off + n]], [base["g"][off:off + n]]
    room = [None if x is None else [torch.zeros(x[0].numel() + 9, dtype=torch.uint8, device=dev).view(x[0].dtype)
                                    if x[0].dtype == torch.float8_e4m3fn else torch.ones(x[0].numel() + 9, device=dev)
                                    ] for x in st]
    if bits == 32:
        for r in room[:2]:
            r[0].zero_()
    sv = [None if x is None else [r[0][off:off + x[0].numel()]] for r, x in zip(room, st)]
    edge = base["p"].clone()
    for t in (1, 2):
        df.adamw_update(whole[0], whole[1], st[0], st[1], t, m_scales=st[2], v_scales=st[3], **HYPER)
        df.adamw_update(views[0], views[1], sv[0], sv[1], t, m_scales=sv[2], v_scales=sv[3], **HYPER)
    assert torch.equal(whole[0][0], views[0][0])
    for a, b in zip(st, sv):
        if a is not None:
            assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8))
    assert torch.equal(base["p"][:off], edge[:off]) and torch.equal(base["p"][off + n:], edge[off + n:])


def test_offsets_past_32_bits(dev):
    """An 8-bit state of a tensor whose byte offsets pass 2^32: its far end equals the same values on their own."""
    n = (1 << 30) + 1000
    p = torch.zeros(n, device=dev)
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    at = n - n % 256 - 1024  # a multiple of 256
    tail = n - at
    p[at:] = torch.randn(tail, device=dev)
    g[at:] = torch.randn(tail, device=dev).bfloat16()
    q, h = [p[at:].clone()], [g[at:].clone()]
    st, s2 = df.adamw_state([p], 8), df.adamw_state(q, 8)
    df.adamw_update([p], [g], st[0], st[1], 1, m_scales=st[2], v_scales=st[3], **HYPER)
    df.adamw_update(q, h, s2[0], s2[1], 1, m_scales=s2[2], v_scales=s2[3], **HYPER)
    assert torch.equal(p[at:], q[0]) and torch.equal(st[2][0][at // 256:], s2[2][0])
    assert torch.equal(st[0][0].view(torch.uint8)[at:], s2[0][0].view(torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_follows_step_and_rate(dev, bits):
    p, g = make([1000, 257], 9, torch.bfloat16)
    P, G = dev_list(p, dev), [t.to(dev) for t in g]
    Q = [t.clone() for t in P]
    a, b = df.adamw_state(P, bits), df.adamw_state(Q, bits)
    step = torch.zeros(1, dtype=torch.int32, device=dev)
    lr = torch.full((1,), 1e-3, device=dev)
    # the same from tensors and from numbers, eagerly
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        df.adamw_update(P, G, a[0], a[1], step, lr=lr, m_scales=a[2], v_scales=a[3])
    for t in range(1, 5):
        rate = 1e-3 * t
        lr.fill_(rate)
        graph.replay()
        df.adamw_update(Q, G, b[0], b[1], t, lr=float(np.float32(rate)), m_scales=b[2], v_scales=b[3])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(P, Q)), t
        for x, y in zip(a, b):
            assert x is None or all(torch.equal(u.view(torch.uint8), w.view(torch.uint8)) for u, w in zip(x, y)), t
        for x in G:
            x.mul_(-0.5)


def test_other_stream(dev):
    p, g = make([3000], 10, torch.float32)
    P, G = dev_list(p, dev), [t.to(dev) for t in g]
    s = torch.cuda.Stream()
    M, V, _, _ = df.adamw_state(P)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        df.adamw_update(P, G, M, V, 1, weight_decay=0.0, **HYPER)
    torch.cuda.current_stream().wait_stream(s)
    assert same(host(P)[0], step32(p[0], g[0].numpy(), 0 * p[0], 0 * p[0], 1, 0.0)[0])


@pytest.mark.parametrize("beta2,t", [(0.95, 100), (0.999, 1), (0.9999, 3)])
@pytest.mark.parametrize("bits", [32, 8])
def test_all_magnitudes_bit_exact(dev, bits, beta2, t):
    """Whole units of values of each size, from subnormal to past 2^20, with zeros of both signs among them."""
    rng = np.random.default_rng(11)
    n = 256 * 4 * 40
    size = np.repeat(np.exp2(np.linspace(-149, 40, n // 256)), 256)
    g = (rng.standard_normal(n) * size).astype(F)
    g[rng.random(n) < 0.05] = 0.0
    g[rng.random(n) < 0.05] = -0.0
    p = (rng.standard_normal(n) * np.exp2(rng.uniform(-40, 10, n))).astype(F)
    p[rng.random(n) < 0.02] = -0.0
    P, G = dev_list([p], dev), dev_list([g], dev)
    M, V, MS, VS = df.adamw_state(P, bits)
    m = v = np.zeros(n, F)
    for k in range(2):
        df.adamw_update(P, G, M, V, t + k, lr=3e-3, beta2=beta2, weight_decay=0.1, m_scales=MS, v_scales=VS)
        p, m, v = step32(p, g, m, v, t + k, 0.1, beta2=beta2)
        assert same(host(P)[0], p), k
        if bits == 32:
            assert same(host(M)[0], m) and same(host(V)[0], v), k
        else:
            (cm, sm), (cv, sv) = keep8(m), keep8(v, root=True)
            assert same(host(M)[0], cm) and same(host(V)[0], cv) and same(host(MS)[0], sm) and same(host(VS)[0], sv), k
            m, v = widen(sm, cm), widen(sv, cv, root=True)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gdt,copy", [(torch.float32, None), (torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)])
def test_lists_larger_than_the_cache(dev, bits, gdt, copy):
    """The same tensors next to one that takes the list past 256 MB: equal bits."""
    sizes = [8192 * 3 + 700, 1025, 40_000]
    p, g = make(sizes, 12, gdt)
    big = 40_000_000
    runs = []
    for extra in (0, big):
        P, G = dev_list(p, dev), [t.to(dev) for t in g]
        if extra:
            P.append(torch.ones(extra, device=dev))
            G.append(torch.full((extra,), 1e-3, dtype=gdt, device=dev))
        M, V, MS, VS = df.adamw_state(P, bits)
        C = None if copy is None else [torch.zeros_like(t, dtype=copy) for t in P]
        for t in (1, 2):
            df.adamw_update(P, G, M, V, t, weight_decay=0.1, m_scales=MS, v_scales=VS, copies=C, **HYPER)
        runs.append([x[:3] for x in (P, M, V, MS, VS, C) if x is not None])
        if extra:  # all values of the filler are alike, and so are their updates
            assert (P[3] == P[3][0]).all() and (bits == 32 or (MS[3] == MS[3][0]).all())
            assert copy is None or (C[3] == P[3][0].to(copy)).all()
    for a, b in zip(*runs):
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("gdt,copy", [(torch.float32, None), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("bits", [32, 8])
def test_views_past_the_cache(dev, bits, gdt, copy):
    """A list past 256 MB of which one tensor, its gradient, states and copy lie at odd elements: equal to plain ones."""
    n, big = 8192 * 2 + 1300, 40_000_000
    p, g = make([n], 13, gdt)
    at = lambda t, k: torch.cat([t.view(torch.uint8).new_zeros(k * t.element_size()), t.view(torch.uint8).reshape(-1),
                                 t.view(torch.uint8).new_zeros(16)])[k * t.element_size():][:t.numel() * t.element_size()].view(t.dtype)
    runs = []
    for k in (0, 1, 3):
        P, G = [at(t, k) for t in dev_list(p, dev)], [at(t.to(dev), k) for t in g]
        st = [None if x is None else [at(x[0], k)] for x in df.adamw_state(P, bits)]
        C = None if copy is None else [at(torch.zeros(n, dtype=copy, device=dev), k)]
        assert P[0].data_ptr() % 16 == 4 * k % 16 and st[0][0].data_ptr() % 16 == (k if bits == 8 else 4 * k) % 16
        fill = torch.ones(big, device=dev)
        more = df.adamw_state([fill], bits)
        args = [P + [fill], G + [torch.zeros(big, dtype=gdt, device=dev)]]
        M, V, MS, VS = (None if x is None else x + y for x, y in zip(st, more))
        copies = None if C is None else C + [torch.zeros(big, dtype=copy, device=dev)]
        for t in (1, 2):
            df.adamw_update(*args, M, V, t, weight_decay=0.1, m_scales=MS, v_scales=VS, copies=copies, **HYPER)
        runs.append([x[0].clone() for x in (P, M, V, MS, VS, copies) if x is not None])
    for other in runs[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(runs[0], other))
