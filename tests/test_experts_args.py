"""Refusals of the experts' products (CPU only: none launches a kernel)."""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import DType

FAKE = 0x1000  # never dereferenced
F32 = int(DType.FLOAT32)


def rows_call(fn, a=FAKE, lda=32, w=FAKE, ldw=32, rows=8, N=32, K=32, experts=4, off=FAKE, s=FAKE, sw=FAKE, dt=F32, out=FAKE,
              ldo=32):
    return getattr(df.lib(), fn)(a, lda, w, ldw, rows, N, K, experts, off, s, sw, dt, out, ldo, None)


@pytest.mark.parametrize("fn", ["df_fp8_experts_fwd", "df_fp8_experts_dx"])
@pytest.mark.parametrize("status,kw", [
    (-1, dict(rows=-1)), (-1, dict(rows=0x7FFFFFFF)), (-1, dict(N=-1, K=-1)), (-1, dict(experts=-1)), (-2, dict(experts=1025)),
    (-2, dict(dt=int(DType.INT8))), (-1, dict(ldo=31)), (-1, dict(off=None)), (-1, dict(s=None)), (-1, dict(sw=None)),
    (-1, dict(out=None)), (-1, dict(a=None)), (-1, dict(w=None)), (-4, dict(lda=24)), (-4, dict(ldw=16)),
    (-4, dict(a=FAKE + 8)), (-4, dict(w=FAKE + 8)), (-2, dict(ldw=1 << 23)), (-4, dict(off=FAKE + 2)), (-4, dict(out=FAKE + 2)),
    (0, dict(rows=0, a=None, out=None)), (0, dict(experts=0, w=None)),
])
def test_rows_refusals(fn, status, kw):
    assert rows_call(fn, **kw) == status
    if status:
        assert fn in df.lib().df_last_error_string().decode()


def dw_call(a=FAKE, lda=16, b=FAKE, ldb=16, rows=8, N=32, K=32, experts=4, off=FAKE, s=FAKE, sx=FAKE, dt=F32, out=FAKE, ldo=32):
    return df.lib().df_fp8_experts_dw(a, lda, b, ldb, rows, N, K, experts, off, s, sx, dt, out, ldo, None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(rows=-1)), (-1, dict(N=-1)), (-1, dict(K=-1)), (-2, dict(experts=2000)), (-2, dict(dt=99)), (-1, dict(ldo=31)),
    (-1, dict(off=None)), (-1, dict(sx=None)), (-1, dict(out=None)), (-1, dict(a=None)), (-4, dict(lda=8)),
    (-4, dict(rows=17)), (-4, dict(b=FAKE + 4)), (-2, dict(lda=1 << 23)), (-1, dict(N=1 << 30, K=1 << 30, ldo=1 << 30)),
    (0, dict(experts=0)), (0, dict(N=0)),
])
def test_dw_refusals(status, kw):
    assert dw_call(**kw) == status
    if status:
        assert "df_fp8_experts_dw" in df.lib().df_last_error_string().decode()


class Fake(torch.Tensor):
    is_cuda = True


def fake(*shape, dtype=torch.uint8):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Fake)


def args(**kw):
    a = dict(x_q=fake(8, 32), w_q=fake(4, 16, 32), offsets=fake(5, dtype=torch.int32), K=32,
             sx=fake(1, dtype=torch.float32), sw=fake(4, dtype=torch.float32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(x_q=torch.zeros(8, 32, dtype=torch.uint8)), "not on a GPU"), (dict(x_q=fake(32)), "dimensions"),
    (dict(w_q=fake(4, 16)), "dimensions"), (dict(x_q=fake(8, 32, dtype=torch.float32)), "codes"),
    (dict(w_q=fake(4, 32, 16).transpose(1, 2)), "codes"), (dict(w_q=fake(8, 16, 32)[::2]), "follow"),
    (dict(offsets=fake(4, dtype=torch.int32)), "offsets"), (dict(offsets=fake(5, dtype=torch.int64)), "offsets"),
    (dict(sx=fake(2, dtype=torch.float32)), "scale"), (dict(sw=fake(3, dtype=torch.float32)), "scales"),
    (dict(K=33), "fewer"), (dict(out=fake(8, 17, dtype=torch.float32)), "out"),
])
def test_python_refusals(kw, word):
    with pytest.raises(ValueError, match=word):
        df.experts_fwd(**args(**kw))


def test_python_refusals_dw():
    ok = dict(dyt_q=fake(16, 16), xt_q=fake(32, 16), offsets=fake(3, dtype=torch.int32), rows=10,
              sdy=fake(1, dtype=torch.float32), sx=fake(1, dtype=torch.float32))
    for kw, word in ((dict(rows=17), "fewer"), (dict(offsets=fake(0, dtype=torch.int32)), "offsets"),
                     (dict(xt_q=fake(2, 2, 2)), "dimensions"), (dict(sx=fake(2, dtype=torch.float32)), "scales"),
                     (dict(out=fake(2, 16, 31, dtype=torch.float32)), "out")):
        with pytest.raises(ValueError, match=word):
            df.experts_dw(**{**ok, **kw})
    for w, word in ((torch.zeros(2, 3), "contiguous"), (torch.zeros(2, 3, 4).transpose(1, 2), "contiguous"),
                    (torch.zeros(2, 3, 4), "not on a GPU")):
        with pytest.raises(ValueError, match=word):
            df.quantize_experts(w)
