"""df_fp8_experts_fwd, _dx and _dw against the products per expert in binary64.

Most tests use codes of small whole numbers and scales that are powers of two:
every partial sum is then a whole number below 2^24 times a power of two, exact
in binary32 whatever the order of the additions, so fp32 outputs have to be
equal and 2-byte outputs equal to the exact value's rounding.  With real data
the bar of an fp32 output is the worst case of a binary32 sum of n products in
any order, each addition off by a step (2 u, for adders that truncate):
2 (n + 8) u sum|a b|.  A 2-byte output comes from the fp8 matrix instructions,
which add products in groups of eight and truncate each to a multiple of 2^-13
of the group's largest: that one is kept, the seven others lose less than
2^-13 of it each, and the groups' largest add up to at most sum|a b|, so
7 * 2^-13 sum|a b| comes on top.
"""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import Fmt

pytestmark = pytest.mark.gpu

U32 = torch.finfo(torch.float32).eps / 2
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def codes(g, dev, shape, fmt, ld, whole=True):
    """uint8 codes [..., ld] (poison past shape[-1] up to the next 16: zeros; beyond: NaN) and their values"""
    if whole:
        v = torch.randint(-8, 9, shape, generator=g, device=dev).float()
        v = v * (v != 9)
    else:
        v = torch.randn(shape, generator=g, device=dev) * 20
    q = v.clamp(-448, 448).to(fmt)
    out = torch.full((*shape[:-1], ld), 0x7F, dtype=torch.uint8, device=dev)
    k = shape[-1]
    out[..., :df.round16(k)] = 0
    out[..., :k] = q.view(torch.uint8)
    return out, q.double()


def bounds(counts):
    b = [0]
    for c in counts:
        b.append(b[-1] + c)
    return b


class Case:
    def __init__(self, dev, counts, K, N, behind=0, seed=0, whole=True, pad=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.b, self.E, self.K, self.N = bounds(counts), len(counts), K, N
        self.rows = self.b[-1] + behind
        self.off = torch.tensor(self.b, dtype=torch.int32, device=dev)
        r16 = df.round16
        R = self.rows
        self.xq, self.x = codes(g, dev, (R, K), E4, r16(K) + pad, whole)
        self.wq, self.w = codes(g, dev, (self.E, N, K), E4, r16(K) + pad, whole)
        self.dyq, self.dy = codes(g, dev, (R, N), E5, r16(N) + pad, whole)
        self.wtq = torch.full((self.E, K, r16(N) + pad), 0x7F, dtype=torch.uint8, device=dev)
        self.wtq[..., :r16(N)] = 0
        self.wtq[..., :N] = self.wq[..., :K].transpose(1, 2)
        # dW: rows of the transposed codes end where they like; what is behind the last expert is NaN codes
        self.xtq = torch.full((K, r16(R) + pad), 0x7F, dtype=torch.uint8, device=dev)
        self.xtq[:, :R] = self.xq[:, :K].t()
        self.dytq = torch.full((N, r16(R) + pad), 0x7F, dtype=torch.uint8, device=dev)
        self.dytq[:, :R] = self.dyq[:, :N].t()
        if behind:
            self.xtq[:, self.b[-1]:] = 0x7F
            self.dytq[:, self.b[-1]:] = 0x7F
        self.sx, self.sdy = torch.tensor([0.25], device=dev), torch.tensor([2.0 ** -7], device=dev)
        self.sw = 2.0 ** -(torch.arange(self.E, device=dev) % 5).float()

    def span(self):
        return [(e, lo, hi) for e, (lo, hi) in enumerate(zip(self.b, self.b[1:]))]


def want(c, which, size=False):
    """the exact product (and, with size, the sum of its terms' magnitudes)"""
    m = (lambda t: t.abs()) if size else (lambda t: t)
    dev = c.off.device
    if which == "dw":
        out = torch.zeros(c.E, c.N, c.K, dtype=torch.float64, device=dev)
        for e, lo, hi in c.span():
            out[e] = m(c.dy[lo:hi]).t() @ m(c.x[lo:hi]) * (c.sdy.double() * c.sx.double())
        return out
    a, w, s = (c.x, c.w.transpose(1, 2), c.sx) if which == "fwd" else (c.dy, c.w, c.sdy)
    out = torch.full((c.rows, w.shape[2]), 777.0, dtype=torch.float64, device=dev)
    for e, lo, hi in c.span():
        out[lo:hi] = m(a[lo:hi]) @ m(w[e]) * (s.double() * c.sw[e].double())
    return out


def run(c, which, dtype, out=None):
    if which == "dw":
        return df.experts_dw(c.dytq, c.xtq, c.off, c.rows, c.sdy, c.sx, out_dtype=dtype, out=out)
    if out is None:
        out = torch.full((c.rows, c.N if which == "fwd" else c.K), 777.0, dtype=dtype, device=c.off.device)
    if which == "fwd":
        return df.experts_fwd(c.xq, c.wq, c.off, c.K, c.sx, c.sw, out=out)
    return df.experts_dx(c.dyq, c.wtq, c.off, c.N, c.sdy, c.sw, out=out)


def check_exact(c, dtypes=(torch.float32, torch.bfloat16, torch.float16), which=("fwd", "dx", "dw")):
    for w in which:
        ref = want(c, w)
        for dt in dtypes:
            got = run(c, w, dt)
            assert torch.equal(got, ref.to(dt)), (w, dt, c.b[:9], c.K, c.N)


COUNTS = [
    [1], [0], [16], [17, 15], [0, 5, 0, 1, 0], [100, 3, 28], [1] * 40, [255, 1, 256, 257], [300, 0, 700],
    [2, 0, 0, 0, 0, 0, 0, 513], [31, 33, 129, 127, 1, 0, 64, 65],
]
SHAPES = [(16, 16), (17, 1), (1, 33), (128, 64), (129, 300), (771, 257), (256, 513)]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "_".join(map(str, c[:9])))
@pytest.mark.parametrize("K,N", SHAPES)
def test_exact(dev, counts, K, N):
    check_exact(Case(dev, counts, K, N, seed=K + len(counts)))


@pytest.mark.parametrize("counts,K,N", [
    ([2048, 1900, 2200, 2044], 640, 768), ([4096], 256, 1600), ([1000, 3000, 0, 96], 1600, 256), ([8] * 64, 1600, 320),
    ([5000, 10, 10, 10], 384, 1040), ([700, 900, 1100, 1300, 1500], 1040, 777),
])
def test_exact_large(dev, counts, K, N):
    """Row counts at which several tiles of an expert are worked on at once."""
    check_exact(Case(dev, counts, K, N, seed=K), dtypes=(torch.float32, torch.bfloat16))


def test_many_experts(dev):
    g = torch.Generator().manual_seed(5)
    counts = torch.randint(0, 5, (1024,), generator=g).tolist()
    check_exact(Case(dev, counts, 64, 48), dtypes=(torch.float32,))
    counts = torch.randint(0, 70, (200,), generator=g).tolist()
    check_exact(Case(dev, counts, 96, 80), dtypes=(torch.bfloat16,))


@pytest.mark.parametrize("counts,behind", [([37, 0, 91], 60), ([0, 0], 33), ([600, 700], 300)])
def test_rows_behind_the_last_expert(dev, counts, behind):
    """Rows that belong to no expert stay as they were, and their codes (NaN here, for dW) reach nothing."""
    c = Case(dev, counts, 200, 144, behind=behind)
    check_exact(c)


def test_neighbours_nan_stays_out(dev):
    """An expert whose codes are all NaN changes no other expert's output."""
    counts = [37, 21, 0, 70, 5]
    c = Case(dev, counts, 100, 60)
    for bad in (0, 1, 3, 4):
        lo, hi = c.b[bad], c.b[bad + 1]
        d = Case(dev, counts, 100, 60)
        d.xtq[:, lo:hi] = 0x7F
        d.dytq[:, lo:hi] = 0x7F
        d.xq[lo:hi] = 0x7F
        for w in ("fwd", "dw"):
            got, ref = run(d, w, torch.float32), want(c, w).float()
            if w == "dw":
                ok = [e for e in range(5) if e != bad]
                assert torch.equal(got[ok], ref[ok]) and got[bad].isnan().all()
            else:
                keep = torch.ones(c.rows, dtype=torch.bool, device=dev)
                keep[lo:hi] = False
                assert torch.equal(got[keep], ref[keep]) and got[~keep].isnan().all()


@pytest.mark.parametrize("counts,K,N", [([90, 0, 300, 11], 777, 640), ([1500, 600, 900], 1600, 512), ([3] * 30, 640, 1600)])
def test_real_data(dev, counts, K, N):
    c = Case(dev, counts, K, N, whole=False)
    for w, n in (("fwd", K), ("dx", N), ("dw", max(counts))):
        ref, size = want(c, w), want(c, w, size=True)
        for dt in (torch.float32, torch.bfloat16, torch.float16):
            got = run(c, w, dt).double()
            f = torch.finfo(dt)
            over = ref.abs() > f.max
            sums = 2 * (n + 8) * U32 + (0 if dt == torch.float32 else 7 * 2.0 ** -13)
            bar = f.eps / 2 * ref.abs() + sums * size + f.smallest_normal * f.eps / 2
            assert ((got - ref).abs()[~over] <= bar[~over]).all(), (w, dt)


def test_every_code(dev):
    """All 256 codes of each format, alone in their sums: fp32 outputs are their values times a power of two."""
    off = torch.tensor([0, 256], dtype=torch.int32, device=dev)
    s = torch.ones(1, device=dev)
    one4, one5 = (torch.tensor([1.0]).to(f).view(torch.uint8).item() for f in (E4, E5))
    for which in ("fwd", "dx", "dw"):
        fa, one = (E4, one4) if which == "fwd" else (E5, one5)
        every = torch.arange(256, dtype=torch.uint8, device=dev)
        a = torch.zeros(256, 16, dtype=torch.uint8, device=dev)
        a[:, 3] = every  # row i: code i of A's format times 1
        w = torch.zeros(1, 256, 16, dtype=torch.uint8, device=dev)
        w[0, :, 3] = one4
        if which == "dw":
            off = torch.tensor([0, 16], dtype=torch.int32, device=dev)
            got = df.experts_dw(a, w[0], off, 16, s, s)[0][:, 0]
            b = torch.zeros(256, 16, dtype=torch.uint8, device=dev)
            b[:, 3] = one5
            other = df.experts_dw(b, a, off, 16, s, s)[0][0]
        else:
            fn = df.experts_fwd if which == "fwd" else df.experts_dx
            got = fn(a, w, off, 16, s, s, out_dtype=torch.float32)[:, 0]
            b = torch.zeros(256, 16, dtype=torch.uint8, device=dev)
            b[:, 3] = one
            other = fn(b, a[None], off, 16, s, s, out_dtype=torch.float32)[0]
        for v, f in ((got, fa), (other, E4)):
            ref = every.view(f).float()
            assert torch.equal(v.isnan(), ref.isnan()) and torch.equal(v.nan_to_num(), ref.nan_to_num())


@pytest.mark.parametrize("counts,K,N", [([33, 95], 100, 52), ([800, 700], 272, 516)])
def test_strided_codes_and_outputs(dev, counts, K, N):
    c = Case(dev, counts, K, N, pad=32)
    check_exact(c)
    for w in ("fwd", "dx"):
        cols = N if w == "fwd" else K
        for extra in (1, 8):
            wide = torch.full((c.rows, cols + extra), 5.0, device=dev)
            run(c, w, torch.float32, out=wide[:, :cols])
            assert torch.equal(wide[:, :cols], want(c, w).float()) and (wide[:, cols:] == 5).all()


def test_wrong_offsets_stay_inside(dev):
    """Offsets out of range or decreasing: in-bounds accesses only (the results mean nothing), and a right call after."""
    c = Case(dev, [40, 30, 50], 64, 48)
    good = c.off.clone()
    for bad in ([-5, 40, 1000, 120], [0, 90, 20, 120], [120, 0, 0, 0], [2 ** 31 - 1] * 4, [-2 ** 31] * 4):
        c.off = torch.tensor(bad, dtype=torch.int64, device=dev).to(torch.int32)
        for w in ("fwd", "dx", "dw"):
            run(c, w, torch.float32)
    torch.cuda.synchronize()
    c.off = good
    check_exact(c, dtypes=(torch.float32,))


def test_quantize_experts(dev):
    g = torch.Generator(device=dev).manual_seed(2)
    for E, N, K in ((3, 40, 96), (5, 37, 51), (1, 16, 16)):
        for dt in (torch.float32, torch.bfloat16, torch.float16):
            w = (torch.randn(E, N, K, generator=g, device=dev) * torch.arange(1, E + 1, device=dev).view(E, 1, 1)).to(dt)
            sc, q, qt = df.quantize_experts(w)
            for e in range(E):
                we = w[e].clone()
                am, s = df.absmax_scale(we, Fmt.E4M3)
                a, b = df.quantize_2d(we, s, Fmt.E4M3, want_qt=True)
                assert sc[e] == s[0] and torch.equal(q[e], a) and torch.equal(qt[e], b)
            assert df.quantize_experts(w, want_qt=False)[2] is None
    for shape in ((0, 4, 8), (2, 0, 8), (2, 4, 0)):
        sc, q, qt = df.quantize_experts(torch.zeros(shape, device=dev))
        assert (sc == 1).all() and q.shape == (*shape[:2], df.round16(shape[2])) and not q.any() and not qt.any()


@pytest.mark.parametrize("counts", [[20, 0, 31, 13], [700, 900, 650]])
def test_graph_follows_offsets(dev, counts):
    """A captured call reads the offsets when it is replayed; two graphs at once."""
    c = Case(dev, counts, 272, 160)
    outs, graphs = [], []
    for _ in range(2):
        o = [run(c, w, torch.float32) for w in ("fwd", "dx", "dw")]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            for w, t in zip(("fwd", "dx", "dw"), o):
                run(c, w, torch.float32, out=t)
        outs.append(o)
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for shift in (0, 7, -11):
        b = bounds(counts)
        b[-2] += shift  # the last two experts share their rows otherwise; offsets stay non-decreasing
        c.b = b
        c.off.copy_(torch.tensor(b, dtype=torch.int32))
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for w, a, d in zip(("fwd", "dx", "dw"), *outs):
            assert torch.equal(a, want(c, w).float()) and torch.equal(d, a), (w, shift)


def test_operands_past_32_bits(dev):
    """Weights of many experts whose byte offsets pass 2^31 and 2^32, and dW's as well."""
    E, N, K = 40, 8192, 16384  # 5.4 GB of codes, dW 10.7 GB in bf16
    w = torch.zeros(E, N, K, dtype=torch.uint8, device=dev)
    one = torch.tensor([1.0], device=dev).to(E4).view(torch.uint8)[0]
    w[E - 1, N - 1] = one  # the last expert's last row is ones
    counts = [1] * E
    off = torch.arange(E + 1, dtype=torch.int32, device=dev)
    x = torch.full((E, K), int(one), dtype=torch.uint8, device=dev)
    s, sw = torch.ones(1, device=dev), torch.ones(E, device=dev)
    y = df.experts_fwd(x, w, off, K, s, sw, out_dtype=torch.float32)
    assert y[E - 1, N - 1] == K and y.sum() == K
    del w
    ldt = df.round16(E)
    half = torch.tensor([1.0], device=dev).to(E5).view(torch.uint8)[0]
    dyt = torch.zeros(N, ldt, dtype=torch.uint8, device=dev)
    dyt[N - 1, :E] = half
    xt = torch.zeros(K, ldt, dtype=torch.uint8, device=dev)
    xt[K - 1, :E] = one
    dw = df.experts_dw(dyt, xt, off, E, s, s, out_dtype=torch.bfloat16)
    assert (dw[:, N - 1, K - 1] == 1).all() and dw[E - 1].sum() == 1 and dw[E // 2].sum() == 1


# per side of the choice of kernel: 32 rows an expert (2-byte outputs), 96 (fp32), 64 output columns, 2048 small tiles of dW;
# few tiles and many, wide and narrow ones
@pytest.mark.parametrize("counts,K,N", [
    ([32, 32, 32], 144, 65), ([33, 33, 33], 144, 65), ([33, 40, 35], 160, 64), ([96] * 3, 272, 200), ([97] * 3, 272, 200),
    ([0, 200, 100, 1], 130, 129), ([64] * 40, 256, 264), ([1] * 70, 192, 160), ([0] * 40 + [7], 260, 300),
    ([300] * 9, 1040, 1300), ([129, 383, 640], 1600, 2000), ([0, 0, 2000], 800, 1600), ([13] * 9, 1200, 1000),
    ([127, 128, 129, 255, 256, 257, 15, 16, 17], 520, 1100),
])
def test_exact_around_the_plan(dev, counts, K, N):
    check_exact(Case(dev, counts, K, N, seed=N), dtypes=(torch.float32, torch.bfloat16))


def test_no_reduction(dev):
    """K of no codes and experts without rows on large tiles: zeros, every row of an expert written."""
    off = torch.tensor([0, 100, 400], dtype=torch.int32, device=dev)
    s, sw = torch.ones(1, device=dev), torch.ones(2, device=dev)
    z = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=dev)
    for dt in (torch.float32, torch.bfloat16):
        y = torch.full((450, 300), 3.0, dtype=dt, device=dev)
        df.experts_fwd(z(450, 16)[:, :0], z(2, 300, 16)[..., :0], off, 0, s, sw, out=y)
        assert (y[:400] == 0).all() and (y[400:] == 3).all()
        dw = df.experts_dw(z(2000, 16)[:, :0], z(2000, 16)[:, :0], off * 0, 0, s, s, out_dtype=dt)
        assert dw.shape == (2, 2000, 2000) and (dw == 0).all()


# sides of the choice by estimated time, and row tiles counted through more
# experts than a wave has lanes, most of them empty
@pytest.mark.parametrize("counts,K,N", [
    ([2000], 1024, 512), ([3000], 1024, 512), ([0] * 64 + [2200] + [0] * 60 + [40, 33] + [0] * 8, 160, 100),
    ([0] * 130 + [2300], 160, 36), ([900, 3, 0, 2, 1], 300, 200), ([1, 2, 0, 3, 900], 300, 200), ([31, 33, 32, 1] * 20, 96, 40),
], ids=lambda v: str(v)[:20])
def test_exact_uneven(dev, counts, K, N):
    check_exact(Case(dev, counts, K, N, seed=N, behind=5), dtypes=(torch.float32, torch.bfloat16))


def test_no_reduction_many_columns(dev):
    """K of no codes, on large tiles in the forward too."""
    off = torch.tensor([0, 100, 400], dtype=torch.int32, device=dev)
    s, sw = torch.ones(1, device=dev), torch.ones(2, device=dev)
    z = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=dev)
    for dt in (torch.float32, torch.bfloat16):
        y = torch.full((450, 12000), 3.0, dtype=dt, device=dev)
        df.experts_fwd(z(450, 16)[:, :0], z(2, 12000, 16)[..., :0], off, 0, s, sw, out=y)
        assert (y[:400] == 0).all() and (y[400:] == 3).all()
