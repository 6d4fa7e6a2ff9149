"""df_rmsnorm_forward, _quantize and _backward against the formulas in binary64, at
the sizes where a row passes from a wave to a block and on to memory, at odd
widths, strides and aliases.

Bars (u = half a step of a type relative to the value, finfo.eps / 2):
  y, dx     one rounding to the type of a binary32 value whose error is a few u32
            of its terms' magnitudes (size): |err| <= u_t |value| + 64 u32 * size.
            rstd's relative error is half that of the mean square (sums of cols / 64
            or fewer terms per lane, then a few: below 32 u32 for these widths) plus
            a few u32.
  codes     rounded once from y in binary32, so off by one step only where y lies
            next to a border between codes: each stands for a value within half a
            step (u_t |y|, or half a least step) and 64 u32 |y| of y.
  dgamma    a column's sum adds rows in groups, fewer than rows / 8 + 64 deep, each
            u32 of the partial sums; its terms carry xh's error (64 u32).
"""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import Fmt

pytestmark = pytest.mark.gpu

E8 = torch.float8_e8m0fnu
U32 = torch.finfo(torch.float32).eps / 2
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
FMAX = {Fmt.E4M3: 448.0, Fmt.E5M2: 57344.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def make(dev, rows, cols, dtype, seed, ld=None, std=1.0, level=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(rows, ld or cols, generator=g, device=dev) * std + level).to(dtype)[:, :cols]


def inputs(dev, rows, cols, dtype, seed=0, pad=0):
    ld = cols + pad
    return dict(x=make(dev, rows, cols, dtype, seed, ld, 1.0, 0.3), r=make(dev, rows, cols, dtype, seed + 1, ld, 0.5),
                gamma=make(dev, 1, cols, dtype, seed + 2, None, 0.2, 1.0)[0].contiguous(),
                dy=make(dev, rows, cols, dtype, seed + 4, ld, 0.1), dr=make(dev, rows, cols, dtype, seed + 5, ld, 0.1))


def forward64(s, gamma, eps):
    s = s.double()
    rstd = (s.square().mean(1) + eps) ** -0.5
    y = s * rstd[:, None]
    return (y if gamma is None else y * gamma.double()), rstd


def check_forward(out, x, r, gamma, eps):
    y, s, rstd = out
    assert torch.equal(s, x if r is None else (x.float() + r.float()).to(x.dtype))
    y64, r64 = forward64(s, gamma, eps)
    assert ((rstd.double() - r64).abs() <= 32 * U32 * r64).all()
    assert ((y.double() - y64).abs() <= half_step(x.dtype) * y64.abs() + 64 * U32 * y64.abs() + tiny(x.dtype)).all()


def check_codes(q, sc, s, rstd, gamma, eps, fmt):
    rows, cols = s.shape
    y64, r64 = forward64(s, gamma, eps)
    assert ((rstd.double() - r64).abs() <= 32 * U32 * r64).all()
    nb = -(-cols // 128)
    pad = torch.nn.functional.pad(y64, (0, nb * 128 - cols)).view(rows, nb, 128)
    most, sv = pad.abs().amax(2), sc.double().t()
    if sc.dtype == E8:  # the least power of two in range, but for an absmax within its error of a border
        at_least, at_most = most * (1 - 64 * U32) / FMAX[fmt], most * (1 + 64 * U32) * 2 / FMAX[fmt]
        ok = (sv >= at_least) & (sv < at_most)
    else:
        ok = (sv - most / FMAX[fmt]).abs() <= 66 * U32 * sv
    assert (ok | ((most == 0) & (sv == 1))).all()
    step = sv.repeat_interleave(128, 1)[:, :cols]
    got = q[:, :cols].double() * step
    least = (2.0 ** -9 if fmt == Fmt.E4M3 else 2.0 ** -16) / 2 * step
    bar = torch.maximum(half_step(q.dtype) * y64.abs() * (1 + 2.0 ** -3), least) + 66 * U32 * y64.abs()
    assert ((got - y64).abs() <= bar).all()
    assert not q[:, cols:].view(torch.uint8).any()


def check_backward(out, dy, x, gamma, rstd, dr):
    dx, dg = out
    d, xs, rs = dy.double(), x.double(), rstd.double()[:, None]
    xh = xs * rs
    g = d if gamma is None else d * gamma.double()
    m = (g * xh).mean(1, keepdim=True)
    want = rs * (g - xh * m)
    size = rs * (g.abs() + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
    if dr is not None:
        want, size = want + dr.double(), size + dr.double().abs()
    assert ((dx.double() - want).abs() <= half_step(x.dtype) * want.abs() + 64 * U32 * size + tiny(x.dtype)).all()
    if dg is not None:
        terms = d * xh
        assert ((dg.double() - terms.sum(0)).abs() <= (x.shape[0] / 8 + 128) * U32 * terms.abs().sum(0) + 1e-37).all()


# a wave's chunks, a block's, memory; odd ends; rows for one launch, many, four at a time
SHAPES = [(1, 1), (1, 768), (2, 3), (5, 7), (3, 9), (16, 127), (64, 128), (33, 257), (7, 771), (9, 1024), (130, 1600),
          (4, 2049), (6, 4100), (3, 8191), (5, 12800), (2, 16385), (3, 40001), (1500, 96), (2100, 771)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_backward(dev, dtype, rows, cols):
    t = inputs(dev, rows, cols, dtype)
    for r, gamma, dr in ((t["r"], t["gamma"], t["dr"]), (None, t["gamma"], None), (t["r"], None, None)):
        out = df.rmsnorm_forward(t["x"], gamma, 1e-5, residual=r)
        check_forward(out, t["x"], r, gamma, 1e-5)
        y, s, rstd = out
        got = df.rmsnorm_backward(t["dy"], s, gamma, rstd, dresidual=dr)
        check_backward(got, t["dy"], s, gamma, rstd, dr)
        again = df.rmsnorm_backward(t["dy"], s, gamma, None, 1e-5, dresidual=dr)
        check_backward(again, t["dy"], s, gamma, forward64(s, gamma, 1e-5)[1], dr)
        assert df.rmsnorm_backward(t["dy"], s, gamma, rstd, sums=False)[1] is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", [E8, torch.float32])
@pytest.mark.parametrize("rows,cols", SHAPES + [(16390, 200)])
def test_quantize(dev, dtype, kind, rows, cols):
    t = inputs(dev, rows, cols, dtype)
    for fmt in Fmt:
        for r, gamma, want_y in ((t["r"], t["gamma"], False), (None, t["gamma"], True), (t["r"], None, True)):
            out = df.rmsnorm_quantize(t["x"], gamma, 1e-5, residual=r, fmt=fmt, want_y=want_y, scale_dtype=kind)
            q, sc, s, rstd = out[:4]
            check_codes(q, sc, s, rstd, gamma, 1e-5, fmt)
            if want_y:
                check_forward((out[4], s, rstd), t["x"], r, gamma, 1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,pad", [(37, 771, 5), (5, 2501, 3), (600, 64, 1)])
def test_strides(dev, dtype, rows, cols, pad):
    t = inputs(dev, rows, cols, dtype, pad=pad)
    out = df.rmsnorm_forward(t["x"], t["gamma"], 1e-5, residual=t["r"])
    check_forward(out, t["x"], t["r"], t["gamma"], 1e-5)
    check_backward(df.rmsnorm_backward(t["dy"], t["x"], t["gamma"], out[2], dresidual=t["dr"]), t["dy"], t["x"], t["gamma"],
                   out[2], t["dr"])
    q, sc, s, rstd = df.rmsnorm_quantize(t["x"], t["gamma"], 1e-5, residual=t["r"])
    check_codes(q, sc, s, rstd, t["gamma"], 1e-5, Fmt.E4M3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(70, 771), (4, 2501), (1300, 520), (3, 20001)])
def test_outputs_over_inputs(dev, dtype, rows, cols):
    """The sum over x or the residual, y over the other, dx over dy or x."""
    t = inputs(dev, rows, cols, dtype)
    y, s, rstd = df.rmsnorm_forward(t["x"], t["gamma"], 1e-5, residual=t["r"])
    dx, dg = df.rmsnorm_backward(t["dy"], s, t["gamma"], rstd, dresidual=t["dr"])
    c = lambda k: t[k].clone()
    dt = int(df._in_dtype(t["x"]))
    for sum_over, y_over in (("x", "r"), ("r", "x")):
        b = {"x": c("x"), "r": c("r")}
        rs = torch.empty_like(rstd)
        df.call("df_rmsnorm_forward", dt, b["x"].data_ptr(), rows, cols, cols, b["r"].data_ptr(), cols,
                b[sum_over].data_ptr(), cols, t["gamma"].data_ptr(), 1e-5, b[y_over].data_ptr(), cols, rs.data_ptr(),
                df._stream())
        assert torch.equal(b[sum_over], s) and torch.equal(b[y_over], y) and torch.equal(rs, rstd)
    for over in ("dy", "x", "dr"):
        b = {"dy": c("dy"), "x": s.clone(), "dr": c("dr")}
        g = torch.empty_like(dg)
        need = df.lib().df_rmsnorm_backward_workspace_bytes(rows, cols)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        df.call("df_rmsnorm_backward", dt, b["dy"].data_ptr(), cols, b["x"].data_ptr(), cols, rows, cols,
                t["gamma"].data_ptr(), rstd.data_ptr(), 1e-5, b["dr"].data_ptr(), cols, b[over].data_ptr(), cols,
                g.data_ptr(), ws.data_ptr(), need, df._stream())
        assert torch.equal(b[over], dx)
        check_backward((dx, g), t["dy"], s, t["gamma"], rstd, t["dr"])


@pytest.mark.parametrize("rows,cols", [(6, 500), (3, 3000), (2, 20000)])
def test_values_that_are_not_finite(dev, rows, cols):
    t = inputs(dev, rows, cols, torch.float32)
    x = t["x"].clone()
    x[0, 1], x[1] = float("nan"), 0.0
    y, s, rstd = df.rmsnorm_forward(x, t["gamma"], 1e-5)
    assert y[0].isnan().all() and rstd[0].isnan() and not y[1].any()
    check_forward((y[1:], s[1:], rstd[1:]), x[1:], None, t["gamma"], 1e-5)
    q, sc, _, _ = df.rmsnorm_quantize(x, t["gamma"], 1e-5)
    assert (q[0, :cols].view(torch.uint8) & 0x7F == 0x7F).all() and not q[0, cols:].view(torch.uint8).any()
    assert (sc[:, 0].float() == 1).all() and (sc[:, 1].float() == 1).all()


def test_no_rows(dev):
    x = torch.empty(0, 24, device=dev)
    assert df.rmsnorm_forward(x)[0].shape == (0, 24)
    assert df.rmsnorm_quantize(x)[0].shape == (0, 32)
    dx, dg = df.rmsnorm_backward(x, x, rstd=x.new_empty(0))
    assert dx.shape == (0, 24) and not dg.any() and dg.shape == (24,)


def test_gradient_by_differences(dev):
    """dx and dgamma against the forward's own differences in binary64's formula."""
    t = inputs(dev, 4, 40, torch.float32)
    x, gamma, dy = t["x"].double().requires_grad_(), t["gamma"].double().requires_grad_(), t["dy"].double()
    loss = lambda a, b: (forward64(a, b, 1e-5)[0] * dy).sum()
    _, _, rstd = df.rmsnorm_forward(t["x"], t["gamma"], 1e-5)
    dx, dg = df.rmsnorm_backward(t["dy"], t["x"], t["gamma"], rstd)
    h = 1e-6
    for i, j in ((0, 0), (1, 17), (3, 39)):
        step = torch.zeros_like(x)
        step[i, j] = h
        num = (loss(x + step, gamma) - loss(x - step, gamma)) / (2 * h)
        assert abs(num - dx[i, j]) <= 1e-5 * dx.abs().max()
        step = torch.zeros_like(gamma)
        step[j] = h
        num = (loss(x, gamma + step) - loss(x, gamma - step)) / (2 * h)
        assert abs(num - dg[j]) <= 1e-5 * dg.abs().max()
