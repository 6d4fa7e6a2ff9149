"""Sizes and strides past 32 bits, which the C interface cannot take, are refused
and not cut to their low half (CPU only: tensors without memory, the library call
recorded)."""
import contextlib

import pytest
import torch

import deepfuse_amd as df

BIG = 1 << 32


class Fake(torch.Tensor):
    """A tensor without memory that says it is on GPU 0."""
    is_cuda = True

    def get_device(self):
        return 0


def fake(*shape, dtype=torch.bfloat16, stride=None):
    n = 1
    for s in shape:
        n *= s
    t = torch.empty(n if stride is None else sum((a - 1) * b for a, b in zip(shape, stride)) + 1, dtype=dtype, device="meta")
    return (t.view(shape) if stride is None else t.as_strided(shape, stride)).as_subclass(Fake)


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(df, "call", lambda *a: made.append(a))
    monkeypatch.setattr(df, "_stream", lambda: 0)
    monkeypatch.setattr(df, "_on", lambda t: contextlib.nullcontext())
    return made


WIDE = dict(stride=(BIG + 8, 1))


@pytest.mark.parametrize("x,kw", [
    (fake(2, 8, **WIDE), {}), (fake(2, 8), dict(residual=fake(2, 8, **WIDE))), (fake(BIG + 2, 4), {}),
    (fake(1 << 31, 1), {}), (fake(1, BIG + 8), {}),
])
def test_layernorm_forward(calls, x, kw):
    with pytest.raises(ValueError, match="32 bits"):
        df.layernorm_forward(x, **kw)
    assert not calls


@pytest.mark.parametrize("dy,x,kw", [
    (fake(2, 8, **WIDE), fake(2, 8), {}), (fake(2, 8), fake(2, 8, **WIDE), {}),
    (fake(2, 8), fake(2, 8), dict(dresidual=fake(2, 8, **WIDE))), (fake(BIG + 2, 4), fake(BIG + 2, 4), {}),
])
def test_layernorm_backward(calls, dy, x, kw):
    with pytest.raises(ValueError, match="32 bits"):
        df.layernorm_backward(dy, x, **kw)
    assert not calls


def u8(*shape, **kw):
    return fake(*shape, dtype=torch.uint8, **kw)


def off(n):
    return fake(n + 1, dtype=torch.int32)


def f32(*shape, **kw):
    return fake(*shape, dtype=torch.float32, **kw)


@pytest.mark.parametrize("x,w,red,kw", [
    (u8(4, 32, stride=(BIG + 32, 1)), u8(2, 16, 32), 32, {}), (u8(4, 32), u8(2, 16, 32, stride=(16 * (BIG + 32), BIG + 32, 1)), 32, {}),
    (u8(BIG + 4, 32), u8(2, 16, 32), 32, {}), (u8(4, 32), u8(2, BIG + 16, 32), 32, {}), (u8(4, BIG + 32), u8(2, 16, BIG + 32), 32, {}),
    (u8(4, BIG + 32), u8(2, 16, BIG + 32), BIG + 32, {}), (u8(4, 32), u8(2, 16, 32), 32, dict(out=f32(4, 16, stride=(BIG + 16, 1)))),
    (u8(4, 32), u8(BIG + 2, 16, 32), 32, {}),
])
@pytest.mark.parametrize("fn", ["experts_fwd", "experts_dx"])
def test_experts_rows(calls, fn, x, w, red, kw):
    E = w.shape[0]
    with pytest.raises(ValueError, match="32 bits"):
        getattr(df, fn)(x, w, off(E), red, f32(1), f32(E), **kw)
    assert not calls


@pytest.mark.parametrize("dyt,xt,rows", [
    (u8(16, 32, stride=(BIG + 32, 1)), u8(8, 32), 20), (u8(16, 32), u8(8, 32, stride=(BIG + 32, 1)), 20),
    (u8(BIG + 16, 32), u8(8, 32), 20), (u8(16, 32), u8(BIG + 8, 32), 20), (u8(16, BIG + 32), u8(8, BIG + 32), BIG + 20),
])
def test_experts_dw(calls, dyt, xt, rows):
    with pytest.raises(ValueError, match="32 bits"):
        df.experts_dw(dyt, xt, off(2), rows, f32(1), f32(1))
    assert not calls


@pytest.mark.parametrize("w", [fake(1, BIG + 1, 2), fake(1, 2, BIG + 1)])
def test_quantize_experts(calls, w):
    with pytest.raises(ValueError, match="32 bits"):
        df.quantize_experts(w)
    assert not calls


def test_what_fits_goes_through(calls):
    most = (1 << 31) - 1
    df.layernorm_forward(fake(2, 8, stride=(most, 1)))
    df.experts_fwd(u8(4, 32, stride=((1 << 31) - 16, 1)), u8(2, 16, 32), off(2), 32, f32(1), f32(2))
    assert calls[0][5] == most and calls[1][2] == (1 << 31) - 16
