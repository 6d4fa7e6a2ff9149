"""df_layernorm_forward and df_layernorm_backward against the formulas in
binary64, at the sizes where a row passes from a wave to a block and on to
memory, at odd widths, strides and aliases, and captured in a graph.

Bars (u = half a step of a type relative to the value, finfo.eps / 2):
  y, dx     one rounding to the type (u_t) of a binary32 value whose error is
            a few u_32 of its terms: |err| <= u_t |value| + 64 u_32 * size, with
            size the sum of the terms' magnitudes (and of what the row's sums
            multiply).  The statistics' relative errors are a few u_32 plus
            those of sums that are added per lane (cols/64 terms or fewer at a
            time): below 32 u_32 for the widths here, less than the 64 counted.
  sums      a column's sum adds rows in order in groups and groups in order:
            fewer than rows/8 + 64 additions deep, each u_32 of the partial
            sums, which stay below sum |term|; its terms carry xh's error
            (64 u_32 as above).
"""
import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu

U32 = torch.finfo(torch.float32).eps / 2
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step among the type's subnormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def make(dev, rows, cols, dtype, seed, ld=None, std=1.0, level=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    base = torch.randn(rows, ld or cols, generator=g, device=dev) * std + level
    return base.to(dtype)[:, :cols]


def inputs(dev, rows, cols, dtype, seed=0, pad=0):
    ld = cols + pad
    return dict(x=make(dev, rows, cols, dtype, seed, ld, 1.0, 0.3), r=make(dev, rows, cols, dtype, seed + 1, ld, 0.5),
                gamma=make(dev, 1, cols, dtype, seed + 2, None, 0.2, 1.0)[0].contiguous(),
                beta=make(dev, 1, cols, dtype, seed + 3, None, 0.2)[0].contiguous(),
                dy=make(dev, rows, cols, dtype, seed + 4, ld, 0.1), dr=make(dev, rows, cols, dtype, seed + 5, ld, 0.1))


def forward64(s, gamma, beta, eps):
    s = s.double()
    mean = s.mean(1)
    var = (s - mean[:, None]).square().mean(1)
    rstd = (var + eps) ** -0.5
    xh = (s - mean[:, None]) * rstd[:, None]
    y, size = xh, (s.abs() + mean.abs()[:, None]) * rstd[:, None]
    if gamma is not None:
        y, size = xh * gamma.double() + beta.double(), size * gamma.double().abs() + beta.double().abs()
    return y, mean, rstd, size


def check_forward(out, x, r, gamma, beta, eps):
    y, s, mean, rstd = out
    want_s = x if r is None else (x.float() + r.float()).to(x.dtype)
    assert torch.equal(s, want_s)
    y64, m64, r64, size = forward64(s, gamma, beta, eps)
    row = s.double().abs().mean(1)
    assert ((mean.double() - m64).abs() <= 32 * U32 * row).all()
    assert ((rstd.double() - r64).abs() <= 64 * U32 * r64 * (1 + (row * r64) ** 2)).all()
    bar = half_step(x.dtype) * y64.abs() + 64 * U32 * size * (1 + (row * r64)[:, None] ** 2) + tiny(x.dtype)
    assert ((y.double() - y64).abs() <= bar).all()


def backward64(dy, x, gamma, mean, rstd, dr):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    xh = (x - mean) * rstd
    g = dy if gamma is None else dy * gamma.double()
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    xs = (x.abs() + mean.abs()) * rstd  # what xh's rounding errors are relative to
    size = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + (xs + xh.abs()) * (g.abs() * xs).mean(1, keepdim=True))
    if dr is not None:
        dx, size = dx + dr.double(), size + dr.double().abs()
    return dx, (dy * xh).sum(0), dy.sum(0), size, (dy.abs() * xs).sum(0), dy.abs().sum(0)


def check_backward(out, dy, x, gamma, mean, rstd, dr, slack=1):
    dx, dg, db = out
    dx64, dg64, db64, size, gs, bs = backward64(dy, x, gamma, mean, rstd, dr)
    assert ((dx.double() - dx64).abs() <= half_step(x.dtype) * dx64.abs() + slack * 64 * U32 * size + tiny(x.dtype)).all()
    deep = x.shape[0] / 8 + 64
    assert dg.dtype == db.dtype == torch.float32
    assert ((dg.double() - dg64).abs() <= (slack * 64 + deep) * U32 * gs + 1e-44).all()
    assert ((db.double() - db64).abs() <= deep * U32 * bs + 1e-44).all()


# widths around: a chunk, a lane's chunk more, a wave's four chunks, blocks of 256 and 512, memory
WIDTHS = [1, 7, 8, 9, 64, 512, 513, 771, 1024, 1600, 2048, 2049, 4096, 5000, 8191, 8192, 16384, 16385, 20001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_forward_and_backward(dev, dtype, cols):
    for rows in (1, 3, 37):
        t = inputs(dev, rows, cols, dtype, seed=cols + rows)
        for r, gamma, beta, dr in ((None, t["gamma"], t["beta"], None), (t["r"], t["gamma"], t["beta"], t["dr"]),
                                   (t["r"], None, None, None)):
            out = df.layernorm_forward(t["x"], gamma, beta, 1e-5, residual=r)
            check_forward(out, t["x"], r, gamma, beta, 1e-5)
            _, s, mean, rstd = out
            check_backward(df.layernorm_backward(t["dy"], s, gamma, mean, rstd, dresidual=dr), t["dy"], s, gamma,
                           mean, rstd, dr)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(0, 64), (5, 0), (2047, 768), (2049, 768), (4100, 200), (16384, 64), (700, 6400),
                                       (300, 12800), (130, 17000)])
def test_many_rows(dev, dtype, rows, cols):
    t = inputs(dev, rows, cols, dtype, seed=rows)
    out = df.layernorm_forward(t["x"], t["gamma"], t["beta"], 1e-5, residual=t["r"])
    if cols:
        check_forward(out, t["x"], t["r"], t["gamma"], t["beta"], 1e-5)
    _, s, mean, rstd = out
    back = df.layernorm_backward(t["dy"], s, t["gamma"], mean, rstd, dresidual=t["dr"])
    if rows == 0:
        assert back[0].shape == (0, cols) and not back[1].any() and not back[2].any()
    elif cols:
        check_backward(back, t["dy"], s, t["gamma"], mean, rstd, t["dr"])
    # no sums: the same dx
    alone = df.layernorm_backward(t["dy"], s, t["gamma"], mean, rstd, dresidual=t["dr"], sums=False)
    assert torch.equal(alone[0], back[0]) and alone[1] is None and alone[2] is None


@pytest.mark.parametrize("rows,cols,over", [(1024, 771, None), (1025, 771, None), (1024, 771, "dy"), (1024, 4200, None),
                                            (1025, 4200, None), (1024, 4200, "s"), (9, 771, None), (8, 771, None)])
def test_both_sides_of_one_launch(dev, rows, cols, over):
    """Rows around the most whose dx and column sums share a launch, and around
    one block's; dx over what the columns' sums read; the same call again."""
    t = inputs(dev, rows, cols, torch.bfloat16, seed=rows + cols)
    s, dy = t["x"], t["dy"]
    _, _, mean, rstd = df.layernorm_forward(s, t["gamma"], t["beta"], 1e-5)
    want = df.layernorm_backward(dy, s, t["gamma"], mean, rstd, dresidual=t["dr"])
    check_backward(want, dy, s, t["gamma"], mean, rstd, t["dr"])
    u = {"dy": dy.clone(), "s": s.clone()}
    dx = torch.empty_like(s) if over is None else u[over]
    dg, db = torch.empty(cols, device=dev), torch.empty(cols, device=dev)
    c_backward(df.DType.BFLOAT16, u["dy"], u["s"], t["gamma"], mean, rstd, t["dr"], dx, dg, db)
    assert torch.equal(dx, want[0]) and torch.equal(dg, want[1]) and torch.equal(db, want[2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,pad", [(771, 5), (1600, 1), (1600, 8), (2500, 3), (17000, 7)])
def test_strided_rows(dev, dtype, cols, pad):
    t = inputs(dev, 19, cols, dtype, seed=cols, pad=pad)
    assert t["x"].stride(0) == cols + pad
    out = df.layernorm_forward(t["x"], t["gamma"], t["beta"], 1e-5, residual=t["r"])
    check_forward(out, t["x"], t["r"], t["gamma"], t["beta"], 1e-5)
    flat = {k: v.contiguous() for k, v in t.items()}
    again = df.layernorm_forward(flat["x"], t["gamma"], t["beta"], 1e-5, residual=flat["r"])
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    _, s, mean, rstd = out
    a = df.layernorm_backward(t["dy"], t["x"], t["gamma"], mean, rstd, dresidual=t["dr"])
    b = df.layernorm_backward(flat["dy"], flat["x"], t["gamma"], mean, rstd, dresidual=flat["dr"])
    assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("cols", [300, 1600, 3000, 17000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_statistics_taken_again(dev, dtype, cols):
    """Without mean and rstd the backward takes them from x: the forward's own values."""
    t = inputs(dev, 65, cols, dtype, seed=cols)
    y, s, mean, rstd = df.layernorm_forward(t["x"], t["gamma"], t["beta"], 1e-3)
    a = df.layernorm_backward(t["dy"], s, t["gamma"], mean, rstd, eps=1e-3)
    b = df.layernorm_backward(t["dy"], s, t["gamma"], eps=1e-3)
    check_backward(b, t["dy"], s, t["gamma"], mean, rstd, None, slack=2)
    for u, v in zip(a, b):  # one rounding of the type apart at most where the statistics' last bits differ
        assert torch.allclose(u.double(), v.double(), rtol=4 * half_step(u.dtype), atol=1e-4)


def test_constant_rows_and_not_finite(dev):
    x = torch.full((4, 1600), 3.0, device=dev)
    x[1, 5] = float("inf")
    x[2, 7] = float("nan")
    g = torch.ones(1600, device=dev)
    y, s, mean, rstd = df.layernorm_forward(x, g, g * 0, 1e-5)
    assert (y[0] == 0).all() and (y[3] == 0).all() and y[1:3].isnan().any(1).all()
    assert rstd[0].item() == pytest.approx(1e-5 ** -0.5, rel=1e-6)
    dx, dg, db = df.layernorm_backward(torch.ones_like(x), x, g, mean, rstd)
    assert dx[0].abs().max() <= 1e-2 * 1600 * U32 * 1e3 and dx[1:3].isnan().any(1).all() and (db == 4).all()


def c_backward(dt, dy, x, gamma, mean, rstd, dr, dx, dg, db):
    rows, cols = x.shape
    ws = torch.empty(int(df.lib().df_layernorm_backward_workspace_bytes(rows, cols)), dtype=torch.uint8, device=x.device)
    df.call("df_layernorm_backward", int(dt), dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), rows, cols,
            gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), 1e-5, dr.data_ptr(), dr.stride(0), dx.data_ptr(),
            dx.stride(0), dg.data_ptr(), db.data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("cols", [515, 771, 1600, 2563, 5000, 17000])
def test_in_place(dev, cols):
    """dx over dy, x or dresidual; sum over x or residual; y over x.  (515, 2563: the row ends in
    a wave's first chunk.)"""
    t = inputs(dev, 40, cols, torch.bfloat16, seed=3)
    y, s, mean, rstd = df.layernorm_forward(t["x"], t["gamma"], t["beta"], 1e-5, residual=t["r"])
    st = torch.cuda.current_stream().cuda_stream
    for over_sum, over_y in (("x", "r"), ("r", "x")):
        u = {k: t[k].clone() for k in ("x", "r")}
        df.call("df_layernorm_forward", int(df.DType.BFLOAT16), u["x"].data_ptr(), 40, cols, cols, u["r"].data_ptr(), cols,
                u[over_sum].data_ptr(), cols, t["gamma"].data_ptr(), t["beta"].data_ptr(), 1e-5, u[over_y].data_ptr(), cols,
                None, None, st)
        assert torch.equal(u[over_sum], s) and torch.equal(u[over_y], y)
    want = df.layernorm_backward(t["dy"], s, t["gamma"], mean, rstd, dresidual=t["dr"])
    for over in ("dy", "s", "dr"):
        u = {"dy": t["dy"].clone(), "s": s.clone(), "dr": t["dr"].clone()}
        dg, db = torch.empty(cols, device=dev), torch.empty(cols, device=dev)
        c_backward(df.DType.BFLOAT16, u["dy"], u["s"], t["gamma"], mean, rstd, u["dr"], u[over], dg, db)
        assert torch.equal(u[over], want[0]) and torch.equal(dg, want[1]) and torch.equal(db, want[2])


def test_gradient_against_differences(dev):
    """d(sum(w * y))/dx along a direction, by central differences of the binary64 formula."""
    t = inputs(dev, 6, 200, torch.float32, seed=9)
    y, s, mean, rstd = df.layernorm_forward(t["x"], t["gamma"], t["beta"], 1e-5)
    dx, dg, db = df.layernorm_backward(t["dy"], s, t["gamma"], mean, rstd)
    f = lambda x, g, b: (forward64(x, g, b, 1e-5)[0] * t["dy"].double()).sum()
    x, g, b, h = s.double(), t["gamma"].double(), t["beta"].double(), 1e-5
    for grad, at, put in ((dx, x, lambda v: (v, g, b)), (dg, g, lambda v: (x, v, b)), (db, b, lambda v: (x, g, v))):
        d = torch.randn_like(at)
        num = (f(*put(at + h * d)) - f(*put(at - h * d))) / (2 * h)
        got = (grad.double() * d).sum()
        # central differences are exact to h^2, about 1e-10 of the terms; binary32 sums to 2^-17 of them
        assert abs(got - num) <= 2 ** -17 * (grad.double() * d).abs().sum() + 1e-6


def test_repeats_and_streams_and_graph(dev):
    t = inputs(dev, 1000, 1600, torch.bfloat16, seed=12)
    step = lambda: df.layernorm_backward(t["dy"], t["x"], t["gamma"], dresidual=t["dr"])
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    # two graphs of the same sizes, replayed at once: each has a workspace of its own
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step())
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        t["dy"].mul_(-1.0)
        eager = step()
        for o in outs:
            for v in o:
                v.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(eager, o)), turn


def test_rows_behind_the_call_stay(dev):
    """Only rows x cols of the outputs are written."""
    st = torch.cuda.current_stream().cuda_stream
    for cols in (771, 1600, 5000):
        t = inputs(dev, 9, cols, torch.float16, seed=4)
        y = torch.full((12, cols + 6), 7.0, dtype=torch.float16, device=dev)
        df.call("df_layernorm_forward", int(df.DType.HALF), t["x"].data_ptr(), 9, cols, cols, None, 0, None, 0,
                t["gamma"].data_ptr(), t["beta"].data_ptr(), 1e-5, y.data_ptr(), cols + 6, None, None, st)
        assert (y[9:] == 7).all() and (y[:, cols:] == 7).all()
        assert torch.equal(y[:9, :cols], df.layernorm_forward(t["x"], t["gamma"], t["beta"])[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_columns(dev, dtype):
    """Statistics over no values are NaN, not what the memory held; no rows give empty ones."""
    torch.full((1 << 16,), 3.0, device=dev)  # freed: what the allocator hands out next
    for rows in (5, 300):
        x = torch.empty(rows, 0, dtype=dtype, device=dev)
        y, s, mean, rstd = df.layernorm_forward(x, residual=x)
        assert y.shape == s.shape == (rows, 0) and mean.shape == rstd.shape == (rows,)
        assert mean.isnan().all() and rstd.isnan().all()
        dx, dg, db = df.layernorm_backward(x, s, None, mean, rstd)
        assert dx.shape == (rows, 0) and dg.shape == db.shape == (0,)
    y, s, mean, rstd = df.layernorm_forward(torch.empty(0, 7, dtype=dtype, device=dev))
    assert y.shape == (0, 7) and mean.shape == rstd.shape == (0,)
