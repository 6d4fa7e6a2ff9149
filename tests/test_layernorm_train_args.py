"""Refusals of the LayerNorm training calls (CPU only: none launches a kernel)."""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import DType

FAKE = 0x1000  # never dereferenced: each call fails its checks first
F32, BF = int(DType.FLOAT32), int(DType.BFLOAT16)


def fwd(dtype=F32, x=FAKE, rows=4, cols=8, ldx=8, res=None, ldr=0, sum=None, lds=0, gamma=FAKE, beta=FAKE, eps=1e-5,
        y=FAKE, ldy=8, mean=None, rstd=None):
    return df.lib().df_layernorm_forward(dtype, x, rows, cols, ldx, res, ldr, sum, lds, gamma, beta, eps, y, ldy, mean, rstd,
                                         None)


def bwd(dtype=F32, dy=FAKE, lddy=8, x=FAKE, ldx=8, rows=4, cols=8, gamma=FAKE, mean=FAKE, rstd=FAKE, eps=1e-5, dr=None,
        lddr=0, dx=FAKE, lddx=8, dg=FAKE, db=FAKE, ws=FAKE, wsb=1 << 20):
    return df.lib().df_layernorm_backward(dtype, dy, lddy, x, ldx, rows, cols, gamma, mean, rstd, eps, dr, lddr, dx, lddx, dg,
                                          db, ws, wsb, None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(rows=-1)), (-1, dict(cols=-1)), (-2, dict(dtype=int(DType.INT8))), (-1, dict(beta=None)), (-1, dict(eps=-1.0)),
    (-1, dict(eps=float("nan"))), (-1, dict(sum=FAKE + 64)), (-1, dict(x=None)), (-1, dict(y=None)), (-1, dict(ldx=7)),
    (-1, dict(ldy=7)), (-1, dict(res=FAKE, ldr=7)), (-1, dict(res=FAKE, ldr=8, sum=FAKE, lds=8, y=FAKE)),
    (-1, dict(res=FAKE, ldr=8, sum=FAKE + 64, lds=7)), (-4, dict(x=FAKE + 2)), (-4, dict(dtype=BF, y=FAKE + 1)),
    (-1, dict(rows=0x7FFFFFFF)), (-1, dict(y=FAKE, ldy=9)), (-1, dict(res=FAKE + 64, ldr=9, sum=FAKE, lds=9, y=FAKE + 128)),
    (-1, dict(res=FAKE + 64, ldr=9, sum=FAKE + 64, lds=8, y=FAKE + 128)), (-4, dict(mean=FAKE + 2)), (0, dict(rows=0, x=None, y=None)), (0, dict(cols=0, ldx=0, ldy=0)),
])
def test_forward_refusals(status, kw):
    assert fwd(**kw) == status
    if status:
        assert "df_layernorm_forward" in df.lib().df_last_error_string().decode()


@pytest.mark.parametrize("status,kw", [
    (-1, dict(rows=-1)), (-1, dict(cols=-1)), (-2, dict(dtype=int(DType.FP8E4M3))), (-1, dict(mean=None)),
    (-1, dict(dg=None)), (-1, dict(eps=-1.0)), (-1, dict(dy=None)), (-1, dict(x=None)), (-1, dict(dx=None)),
    (-1, dict(cols=0x7FFFFFFF, lddy=0x7FFFFFFF)), (-1, dict(dx=FAKE, lddx=9)), (-1, dict(dr=FAKE, lddr=9)),
    (-1, dict(lddy=7)), (-1, dict(ldx=0)), (-1, dict(lddx=7)), (-1, dict(dr=FAKE, lddr=7)), (-4, dict(dy=FAKE + 2)),
    (-4, dict(dg=FAKE + 1)), (-5, dict(ws=None)), (-5, dict(ws=FAKE + 8)), (-5, dict(wsb=4 * 8 * 8 - 1)),
    (0, dict(cols=0, dy=None, x=None, dx=None, ws=None, wsb=0)),
])
def test_backward_refusals(status, kw):
    assert bwd(**kw) == status
    if status:
        assert "df_layernorm_backward" in df.lib().df_last_error_string().decode()


def test_workspace_sizes():
    need = df.lib().df_layernorm_backward_workspace_bytes
    assert need(0, 5) == need(5, 0) == need(-1, 5) == 0
    assert need(4, 8) == 4 * 2 * 8 * 4 + 4 * 8
    assert need(16384, 1600) == 512 * 2 * 1600 * 4 + 16384 * 8


def test_python_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="not on a GPU"):
        df.layernorm_forward(x)
    with pytest.raises(ValueError, match="dimensions"):
        df.layernorm_forward(torch.zeros(4, 8, 2))
    with pytest.raises(ValueError, match="not on a GPU"):
        df.layernorm_backward(x, x)


class Fake(torch.Tensor):
    """A host tensor that says it is on a GPU: for checks that end before any launch."""
    is_cuda = True


@pytest.mark.parametrize("kw,word", [
    (dict(gamma=torch.zeros(7)), "gamma"), (dict(gamma=torch.zeros(8, dtype=torch.bfloat16)), "gamma"),
    (dict(residual=torch.zeros(4, 7)), "residual"), (dict(residual=torch.zeros(1, 8).expand(4, 8)), "strides"),
    (dict(beta=torch.zeros(16)[::2]), "beta"),
])
def test_python_shapes(kw, word):
    as_fake = lambda t: t.as_subclass(Fake)
    with pytest.raises(ValueError, match=word):
        df.layernorm_forward(as_fake(torch.zeros(4, 8)), **{k: as_fake(v) for k, v in kw.items()})
    with pytest.raises(ValueError, match="strides"):
        df.layernorm_forward(as_fake(torch.zeros(8, 4).t()))
