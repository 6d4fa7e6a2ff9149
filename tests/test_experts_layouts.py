"""Leading dimensions that the experts' products hand on: a dimension of one has
an arbitrary stride, on which torch still calls a tensor contiguous (CPU only:
the library call is recorded, not made)."""
import contextlib

import pytest
import torch

import deepfuse_amd as df


class Fake(torch.Tensor):
    """A host tensor that says it is on GPU 0."""
    is_cuda = True

    def get_device(self):
        return 0


def fake(*shape, dtype=torch.uint8):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Fake)


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(df, "call", lambda *a: made.append(a))
    monkeypatch.setattr(df, "_stream", lambda: 0)
    monkeypatch.setattr(df, "_on", lambda t: contextlib.nullcontext())
    return made


def off(n):
    return fake(n + 1, dtype=torch.int32)


def f32(n):
    return fake(n, dtype=torch.float32)


def rows_call(fn, x, w, red):
    E = w.shape[0]
    return getattr(df, fn)(x, w, off(E), red, f32(1), f32(E))


# codes [1, 32] and their like with every stride that a dimension of one may have, and the leading dimension they mean
ONE_ROW = [
    (lambda: fake(1, 32), 32), (lambda: fake(32, 1).t(), 32), (lambda: fake(4, 64)[2:3, :32], 32),
    (lambda: fake(4, 48)[2:3, :20], 48), (lambda: fake(32).as_strided((1, 32), (7, 1)), 32),
    (lambda: fake(32).as_strided((1, 32), (0, 1)), 32),
]


@pytest.mark.parametrize("fn", ["experts_fwd", "experts_dx"])
@pytest.mark.parametrize("make,ld", ONE_ROW)
def test_one_row(calls, fn, make, ld):
    x = make()
    rows_call(fn, x, fake(3, 16, 32), 20)
    assert calls[0][2] == ld and calls[0][4] == 32 and calls[0][5] == 1


@pytest.mark.parametrize("make,ld", ONE_ROW)
def test_one_row_dw(calls, make, ld):
    t = make()
    df.experts_dw(t, fake(5, 32), off(2), 20, f32(1), f32(1))
    df.experts_dw(fake(5, 32), t, off(2), 20, f32(1), f32(1))
    assert calls[0][2] == ld and calls[0][4] == 32 and calls[1][2] == 32 and calls[1][4] == ld


@pytest.mark.parametrize("fn", ["experts_fwd", "experts_dx"])
@pytest.mark.parametrize("make,ld", [
    (lambda: fake(4, 1, 32), 32), (lambda: fake(1, 4, 32).transpose(0, 1), 32), (lambda: fake(4, 64)[:, None, :32], 64),
    (lambda: fake(4, 5, 32)[:, 2:3], 160), (lambda: fake(1, 4, 64)[..., :32].transpose(0, 1), 64),
    (lambda: fake(1, 1, 32), 32), (lambda: fake(32, 1, 1).permute(1, 2, 0), 32), (lambda: fake(4, 8, 32), 32),
    (lambda: fake(4, 8, 64)[..., :32], 64), (lambda: fake(1, 8, 64)[..., :32], 64),
])
def test_one_column(calls, fn, make, ld):
    """Weights of one output column: the step from expert to expert is the leading dimension."""
    w = make()
    rows_call(fn, fake(8, 32), w, 32)
    assert calls[0][2] == 32 and calls[0][4] == ld
    n, k = calls[0][6:8] if fn == "experts_fwd" else calls[0][7:5:-1]
    assert (n, k) == (w.shape[1], 32)


def test_experts_apart(calls):
    for w in (fake(4, 6, 32)[:, ::2], fake(4, 6, 32)[:, :3], fake(8, 6, 32)[::2]):
        if w.stride(0) != w.shape[1] * w.stride(1):
            with pytest.raises(ValueError, match="follow"):
                rows_call("experts_fwd", fake(8, 32), w, 32)
    assert not calls


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 4, 8), (3, 5, 7), (1, 4, 8)])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_weights_at_any_element(calls, dtype, shape, offset):
    """Experts' weights that start at any element are quantized from 16-byte boundaries, with their values."""
    n = shape[0] * shape[1] * shape[2]
    base = torch.arange(64 + n).to(dtype)
    start = -(base.data_ptr() % 16) // base.element_size() % 8 + offset
    w = base[start:start + n].view(shape).as_subclass(Fake)
    df.quantize_experts(w)
    ptrs = [list(c[3]) for c in calls if c[0] == "df_quantize_2d_batch"]
    ptrs = ptrs[0] if ptrs else [c[2] for c in calls]
    assert len(ptrs) == shape[0] and all(p % 16 == 0 for p in ptrs)
