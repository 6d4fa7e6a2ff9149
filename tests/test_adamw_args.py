"""Refusals of df_adamw_update, df_grad_norm and their Python forms (CPU only:
none launches a kernel)."""
import ctypes
import warnings

import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import DType

P = ctypes.c_void_p
FAKE = 0x1000  # never dereferenced
F32, BF, E4 = int(DType.FLOAT32), int(DType.BFLOAT16), int(DType.FP8E4M3)


def one(v=FAKE):
    return (P * 1)(v)


def call(count=1, n=4, p=one(), gt=F32, g=one(), st=F32, m=one(), v=one(), ms=None, vs=None, ct=0, copies=None, t=1, lr=None,
         step=None, norm=None, am=None):
    sizes = (ctypes.c_int64 * 1)(n)
    return df.lib().df_adamw_update(count, sizes, p, gt, g, st, m, v, ms, vs, ct, copies, 1e-3, 0.9, 0.99, 1e-8, None, t, lr,
                                    step, norm, 0.0, am, None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(count=-1)), (-1, dict(n=-4)), (-1, dict(p=None)), (-1, dict(p=one(None))), (-1, dict(g=one(None))),
    (-1, dict(v=None)), (-2, dict(gt=int(DType.INT8))), (-2, dict(st=BF)), (-2, dict(st=int(DType.FP8E5M2))),
    (-2, dict(copies=one(), ct=F32)), (-1, dict(copies=one(None), ct=BF)), (-1, dict(st=E4)),
    (-1, dict(st=E4, ms=one(None), vs=one())), (-1, dict(t=0)), (-4, dict(p=one(FAKE + 2))), (-4, dict(gt=BF, g=one(FAKE + 1))),
    (-4, dict(m=one(FAKE + 1))), (-4, dict(st=E4, m=one(FAKE + 1), ms=one(FAKE + 2), vs=one())), (-4, dict(lr=FAKE + 1)),
    (-4, dict(step=FAKE + 2)), (-4, dict(copies=one(FAKE + 1), ct=BF)), (-1, dict(n=1 << 62)), (0, dict(count=0)),
    (0, dict(n=0, p=one(None), g=one(None), m=one(None), v=one(None))),
])
def test_refusals(status, kw):
    assert call(**kw) == status
    if status:
        assert "df_adamw_update" in df.lib().df_last_error_string().decode()


def test_scale_count():
    assert [df.lib().df_adamw_scale_count(n) for n in (-1, 0, 1, 256, 257, 1 << 33)] == [0, 0, 1, 1, 2, 1 << 25]


def test_grad_norm_refusals():
    sizes = (ctypes.c_int64 * 1)(4)
    g = df.lib().df_grad_norm
    assert g(int(DType.INT8), one(), sizes, 1, FAKE, FAKE, 64, None) == -2
    assert g(BF, one(FAKE + 1), sizes, 1, FAKE, FAKE, 64, None) == -4
    assert g(BF, one(None), sizes, 1, FAKE, FAKE, 64, None) == -1
    assert g(BF, one(FAKE + 2), sizes, 1, FAKE, FAKE, 4, None) == -5
    assert g(F32, one(FAKE + 4), sizes, 1, FAKE, FAKE, 64, None) == -4  # the fp32 lists keep their 16 bytes
    assert g(BF, one(), sizes, -1, FAKE, FAKE, 64, None) == -1


class Fake(torch.Tensor):
    is_cuda = True


def fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Fake)


def test_python_refusals():
    p, g = [torch.zeros(4)], [torch.zeros(4)]
    with pytest.raises(ValueError, match="a GPU"):
        df.adamw_update(p, g, g, g, 1)
    with pytest.raises(ValueError, match="bits"):
        df.adamw_state(p, 16)
    ok = lambda: [fake(4)]
    for bad, word in ((dict(grads=[fake(5)]), "grads"), (dict(ms=[]), "ms"), (dict(vs=[fake(4, dtype=torch.bfloat16)]), "vs"),
                      (dict(m_scales=ok()), "go together"), (dict(params=[fake(4, 4).t()]), "params"),
                      (dict(weight_decay=[0.1, 0.2]), "weight decays"), (dict(timestep=fake(1)), "timestep"),
                      (dict(lr=fake(2)), "lr"), (dict(absmax=fake(0)), "absmax"), (dict(clip_norm=fake(2)), "clip_norm"),
                      (dict(copies=[fake(3, dtype=torch.bfloat16)]), "copies")):
        kw = dict(params=ok(), grads=ok(), ms=ok(), vs=ok(), timestep=1)
        kw.update(bad)
        with pytest.raises(ValueError, match=word):
            df.adamw_update(**kw)
    with pytest.raises(TypeError, match="copies"):
        df.adamw_update(ok(), ok(), ok(), ok(), 1, copies=ok())
    t = fake(4)
    with pytest.raises(ValueError, match="twice"):
        df.adamw_update([t, t], [fake(4), fake(4)], [fake(4), fake(4)], [fake(4), fake(4)], 1)
    df.adamw_update([], [], [], [], 1)
    with pytest.raises(TypeError, match="not clipped"):
        df.grad_norm([torch.zeros(4, dtype=torch.bfloat16)], clip=1.0)


def test_clip_needs_a_device_norm_and_a_limit():
    """A number in the norm's place would clip nothing, a norm without a limit would zero every gradient."""
    ok = lambda: [fake(4)]
    for norm in (50.0, 1, torch.nn.Identity(), [fake(1)]):
        with pytest.raises(TypeError, match="clip_norm"):
            df.adamw_update(ok(), ok(), ok(), ok(), 1, clip_norm=norm, max_norm=1.0)
    for kw in (dict(), dict(max_norm=0.0), dict(max_norm=-1.0), dict(max_norm=float("nan"))):
        with pytest.raises(ValueError, match="max_norm"):
            df.adamw_update(ok(), ok(), ok(), ok(), 1, clip_norm=fake(1), **kw)


def test_dither_refusals():
    sizes = (ctypes.c_int64 * 1)(4)
    f = lambda st=E4, n=sizes, t=1, ms=one(): df.lib().df_adamw_update_dithered(
        1, n, one(), F32, one(), st, one(), one(), ms, one(), 0, None, 1e-3, 0.9, 0.99, 1e-8, None, t, None, None, None, 0.0,
        None, 7, None)
    assert f(st=F32) == -2 and f(st=BF) == -2 and f(t=0) == -1 and f(ms=None) == -1 and f(n=(ctypes.c_int64 * 1)(-1)) == -1
    assert "df_adamw_update_dithered" in df.lib().df_last_error_string().decode()
    assert f(n=(ctypes.c_int64 * 1)(0)) == 0
    ok = lambda: [fake(4)]
    with pytest.raises(ValueError, match="dither"):
        df.adamw_update(ok(), ok(), ok(), ok(), 1, dither=0)


def test_nearest_warns_once(monkeypatch):
    """8-bit states without dither: said once; 32-bit ones and dithered ones say nothing."""
    monkeypatch.setattr(df, "_nearest_told", False)
    codes = lambda: [torch.zeros(4).to(torch.float8_e4m3fn).as_subclass(Fake)]
    ok = lambda: [fake(4)]
    bad = dict(clip_norm=1.0)  # ends the call before the library
    run = lambda **kw: pytest.raises(TypeError, df.adamw_update, ok(), ok(), codes(), codes(), 1, m_scales=[fake(1)],
                                     v_scales=[fake(1)], **bad, **kw)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        run(dither=0)
        pytest.raises(TypeError, df.adamw_update, ok(), ok(), ok(), ok(), 1, **bad)
    with pytest.warns(UserWarning, match="dither"):
        run()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        run()
