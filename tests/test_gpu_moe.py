"""df_moe_layer against its definition in binary64: choices, weights and outputs, for
one token and up to 64, every activation and type, odd sizes, experts that get all
tokens or none, ties, masked and missing experts, strides, and wide values.

Bars: ids are equal.  weights: an exponential's error (2 u32 of its value and of its
argument's rounding, |l - most| u32) over a sum of up to 256 such: 64 u32 (1 + |l -
most|), and below 2^-126, where binary32 has steps of 2^-149, one step each for the
exponential and the quotient.  y: with S2 = sum over choices of weight * sum |W2| * |h| and E the error of h
below, |err| <= u_t |y| + 2^-16 S2 (the two bf16 parts of h, 2^-17 each at most, and
the binary32 sums, fewer than 2^14 terms of 2^-24 / 2, in blocks) + sum weight * sum
|W2| E; h's error is that of its sums, S1 (K + 64) u32 with S1 = sum |W1| |x|, through
an activation whose slope is below 1.2, times the other factor, and 16 u32 of h.
"""
import math

import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu

E8 = torch.float8_e8m0fnu
U32 = torch.finfo(torch.float32).eps / 2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gelu(v):
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))


def values(q, s, cols):
    return q[:, :cols].double() * s.double().t().repeat_interleave(128, 1)[:, :cols]


def weights(dev, E, R, C, kind, g, std=None):
    w = torch.randn(E, R, C, generator=g, device=dev) * (std or C ** -0.5)
    w *= torch.exp(torch.randn(E, R, 1, generator=g, device=dev))
    return df.quantize_experts_blocks(w, scale_dtype=kind)


def make(dev, T, E, H, N, act="swiglu", dtype=torch.bfloat16, kind=E8, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    w1, s1 = weights(dev, E, N if act == "gelu" else 2 * N, H, kind, g)
    w2, s2 = weights(dev, E, H, N, kind, g)
    x = torch.randn(T, H, generator=g, device=dev).to(dtype)
    return x, torch.randn(T, E, generator=g, device=dev), w1, s1, w2, s2


def choose(logits, top, renormalize):
    l = logits.double()
    l = torch.where(l.isnan(), -math.inf, l)
    ids = torch.argsort(-l, dim=1, stable=True)[:, :top]
    best = l.gather(1, ids)
    ids = torch.where(best == -math.inf, -1, ids)
    most = best[:, :1]
    part = lambda v: torch.where(v == most, 1.0, torch.exp(v - most))
    share = torch.where(ids >= 0, part(best), 0.0)
    total = share if renormalize else torch.where(l == -math.inf, 0.0, part(l))
    return ids, torch.where(ids >= 0, share / total.sum(1, keepdim=True), 0.0), torch.where(
        best.isfinite() & most.isfinite(), (best - most).abs(), 0.0)  # (an infinity is chosen alone, or shares alike)


def check(out, x, logits, w1, s1, w2, s2, top, act, renormalize=True):
    y, ids, wt = out
    T, H = x.shape
    N = w1.shape[1] // (1 if act == "gelu" else 2)
    want_ids, want_w, far = choose(logits, top, renormalize)
    assert ids.dtype == torch.int32 and torch.equal(ids.long(), want_ids)
    ok = (wt.double() - want_w).abs() <= 64 * U32 * want_w * (1 + far) + 2.0 ** -148
    assert (ok | (want_ids < 0) & (wt == 0)).all()
    yy, bar = (torch.zeros(T, H, dtype=torch.float64, device=x.device) for _ in range(2))
    for e in range(w1.shape[0]):
        who, place = torch.where(ids == e)
        if not len(who):
            continue
        a, b = values(w1[e], s1[e], H), values(w2[e], s2[e], N)
        xe = x[who].double()
        h, size = xe @ a.t(), (xe.abs() @ a.abs().t()) * (H + 64) * U32
        if act == "gelu":
            v, err = gelu(h), 1.2 * size
        else:
            f = gelu if act == "geglu" else lambda u: u * torch.sigmoid(u)
            v = f(h[:, :N]) * h[:, N:]
            err = 1.2 * size[:, :N] * (h[:, N:].abs() + size[:, N:]) + f(h[:, :N]).abs() * size[:, N:]
        err = err + 16 * U32 * v.abs()
        w = wt.double()[who, place][:, None]
        yy[who] += w * (v @ b.t())
        bar[who] += w * ((2.0 ** -16 * v.abs() + err) @ b.abs().t())
    bar += half_step(x.dtype) * yy.abs() + torch.finfo(x.dtype).smallest_normal
    assert ((y.double() - yy).abs() <= bar).all()


SIZES = [(1, 4, 2, 64, 64), (1, 32, 2, 1600, 1600), (1, 7, 7, 771, 515), (1, 256, 16, 100, 30), (2, 3, 1, 17, 5),
         (2, 8, 2, 1, 1), (3, 5, 2, 130, 129), (16, 2, 1, 256, 128), (17, 2, 2, 300, 200), (33, 64, 6, 257, 260),
         (48, 32, 2, 1600, 800), (64, 4, 2, 96, 1000), (64, 1, 1, 200, 72), (64, 200, 16, 48, 33), (5, 32, 8, 8, 300)]


@pytest.mark.parametrize("act", ["swiglu", "geglu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [E8, torch.float32])
@pytest.mark.parametrize("T,E,top,H,N", SIZES)
def test_sizes(dev, T, E, top, H, N, kind, dtype, act):
    t = make(dev, T, E, H, N, act, dtype, kind)
    check(df.moe_layer(*t, top, activation=act), *t, top, act)


@pytest.mark.parametrize("T", [1, 2, 40])
@pytest.mark.parametrize("logits_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renormalize", [True, False])
def test_routing(dev, T, logits_dtype, renormalize):
    """Ties, signed zeros, infinities, NaN, experts that cannot be chosen."""
    x, logits, *w = make(dev, T, 70, 130, 40)
    logits = logits.to(logits_dtype)
    inf, nan = math.inf, math.nan
    rows = [torch.zeros(70), torch.full((70,), -inf), torch.full((70,), nan), torch.arange(70) % 3 * 1.0,
            torch.where(torch.arange(70) % 2 == 0, 0.0, -0.0), torch.where(torch.arange(70) == 69, 1.0, -inf),
            torch.where(torch.arange(70) % 30 == 5, inf, 1.0), torch.where(torch.arange(70) < 68, nan, -60000.0)]
    for k, row in enumerate(rows):
        l = logits.clone()
        l[k % T] = row.to(logits_dtype)
        for top in (1, 4, 16):
            out = df.moe_layer(x, l, *w, top, renormalize=renormalize)
            check(out, x, l, *w, top, "swiglu", renormalize)
            if k in (1, 2):
                assert (out[1][k % T] == -1).all() and not out[0][k % T].any()


@pytest.mark.parametrize("kind", [E8, torch.float32])
@pytest.mark.parametrize("T,N", [(1, 1200), (2, 1200), (1, 4100)])
def test_few_tokens_in_shares(dev, T, N, kind):
    """So many steps that blocks share W2's columns, for one token (whose routing is no
    launch of its own) too; the blocks' counts start anew in each call."""
    t = make(dev, T, 16, 100, N, "swiglu", torch.bfloat16, kind)
    first = df.moe_layer(*t, 16)
    check(first, *t, 16, "swiglu")
    assert all(torch.equal(a, b) for a, b in zip(first, df.moe_layer(*t, 16)))


@pytest.mark.parametrize("T", [1, 16, 64])
def test_all_tokens_to_one_expert(dev, T):
    x, logits, *w = make(dev, T, 16, 200, 150)
    logits[:, 11] += 100
    out = df.moe_layer(x, logits, *w, 3)
    assert (out[1][:, 0] == 11).all()
    check(out, x, logits, *w, 3, "swiglu")


@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("off,pad", [(1, 0), (0, 3), (5, 6)])
def test_strides_and_addresses(dev, T, off, pad):
    for H in (3, 131, 256):
        x, logits, *w = make(dev, T, 6, H, 70)
        wide = torch.full((T, off + H + pad), math.nan, dtype=x.dtype, device=dev)
        wide[:, off:off + H] = x
        lw = torch.full((T, off + 6 + pad), 1e9, device=dev)
        lw[:, off:off + 6] = logits
        got = df.moe_layer(wide[:, off:off + H], lw[:, off:off + 6], *w, 2)
        want = df.moe_layer(x, logits, *w, 2)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("T", [1, 5])
def test_values_that_are_not_finite(dev, T):
    """A NaN or an infinity of one token stays its own."""
    x, logits, *w = make(dev, T + 1, 4, 150, 64)
    clean = df.moe_layer(x, logits, *w, 2)[0]
    x[T, 149] = math.nan
    y = df.moe_layer(x, logits, *w, 2)[0]
    assert torch.equal(y[:T], clean[:T]) and y[T].isnan().all()


def test_inner_values_beyond_the_types_range(dev):
    """float16 inputs whose inner values pass 65504."""
    g = torch.Generator(device=dev).manual_seed(3)
    H, N = 256, 128
    w1, s1 = weights(dev, 2, 2 * N, H, E8, g, std=1.0)
    w2, s2 = weights(dev, 2, H, N, E8, g, std=1e-4)
    x = (torch.randn(3, H, generator=g, device=dev) * 20).to(torch.float16)
    logits = torch.randn(3, 2, generator=g, device=dev)
    out = df.moe_layer(x, logits, w1, s1, w2, s2, 2)
    check(out, x, logits, w1, s1, w2, s2, 2, "swiglu")
    assert out[0].isfinite().all()


@pytest.mark.parametrize("T", [1, 3, 50])
def test_same_call_same_bits(dev, T):
    t = make(dev, T, 12, 640, 300)
    first = df.moe_layer(*t, 4)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(df.moe_layer(*t, 4), first))


def test_no_tokens(dev):
    y, ids, wt = df.moe_layer(*make(dev, 0, 4, 32, 16), 2)
    assert y.shape == (0, 32) and ids.shape == wt.shape == (0, 2)
