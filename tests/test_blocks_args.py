"""Refusals of the calls with a scale per 128 values, the RMS norm and the experts'
layer (CPU only: none launches a kernel)."""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import DType

FAKE = 0x1000  # never dereferenced: each call fails its checks first
F32, BF, F16, I8 = (int(d) for d in (DType.FLOAT32, DType.BFLOAT16, DType.HALF, DType.INT8))
E8, SF = 1, 0  # df_scale_kind


def refused(status, fn, rc):
    assert rc == status
    if status:
        assert fn in df.lib().df_last_error_string().decode()


def quantize(dtype=BF, x=FAKE, rows=4, cols=40, ldx=40, fmt=0, kind=E8, square=0, q=FAKE, ldq=48, s=FAKE, lds=16, qt=FAKE,
             ldqt=16, st=FAKE, ldst=48):
    return df.lib().df_quantize_blocks(dtype, x, rows, cols, ldx, fmt, kind, square, q, ldq, s, lds, qt, ldqt, st, ldst, None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(rows=-1)), (-1, dict(cols=-1)), (-1, dict(rows=128 * 65535 + 1)), (-2, dict(dtype=I8)), (-1, dict(fmt=2)),
    (-1, dict(kind=2)), (-1, dict(q=None, qt=None)), (-1, dict(s=None)), (-1, dict(st=None)), (-1, dict(x=None)),
    (-1, dict(ldx=39)), (-4, dict(x=FAKE + 1)), (-4, dict(dtype=F32, x=FAKE + 2)), (-4, dict(ldq=40)), (-4, dict(ldq=32)),
    (-4, dict(q=FAKE + 8)), (-4, dict(ldqt=20)), (-4, dict(rows=20, lds=32, ldqt=16)), (-4, dict(qt=FAKE + 4)),
    (-4, dict(lds=8)), (-4, dict(lds=24)), (-4, dict(s=FAKE + 4)), (-4, dict(ldst=32)), (-4, dict(st=FAKE + 8)),
    (-4, dict(kind=SF, lds=6)), (-4, dict(kind=SF, ldst=42)), (0, dict(rows=0, x=None)), (0, dict(cols=0, x=None)),
])
def test_quantize_refusals(status, kw):
    refused(status, "df_quantize_blocks", quantize(**kw))


def gemm(fmt=0, A=FAKE, lda=48, B=FAKE, ldb=48, M=4, N=5, K=40, kind=E8, sa=FAKE, ldsa=16, sb=FAKE, ldsb=16, bdt=F32,
         bias=None, cdt=BF, C=FAKE, ldc=5):
    return df.lib().df_fp8_gemm_blocks(fmt, A, lda, B, ldb, M, N, K, kind, sa, ldsa, sb, ldsb, bdt, bias, cdt, C, ldc, None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(M=-1)), (-1, dict(N=-1)), (-1, dict(K=-1)), (-1, dict(fmt=2)), (-1, dict(kind=5)), (-2, dict(cdt=I8)),
    (-2, dict(bias=FAKE, bdt=I8)), (-1, dict(C=None)), (-1, dict(ldc=4)), (-4, dict(C=FAKE + 1)), (-4, dict(cdt=F32, C=FAKE + 2)),
    (-4, dict(bias=FAKE + 2)), (-1, dict(A=None)), (-1, dict(B=None)), (-1, dict(sa=None)), (-1, dict(sb=None)),
    (-4, dict(lda=40)), (-4, dict(ldb=32)), (-4, dict(A=FAKE + 8)), (-4, dict(B=FAKE + 1)), (-4, dict(ldsa=8)),
    (-4, dict(ldsb=4)), (-4, dict(kind=SF, ldsa=6)), (-4, dict(sa=FAKE + 4)), (-4, dict(sb=FAKE + 8)),
    (-2, dict(lda=1 << 23)), (-2, dict(K=1 << 20, lda=1 << 20, ldb=1 << 20, ldsa=1 << 30, ldsb=16)),
    (-2, dict(M=1 << 18, N=1 << 18, ldc=1 << 18)), (0, dict(M=0, A=None, C=None)), (0, dict(N=0, B=None, C=None)),
])
def test_gemm_refusals(status, kw):
    refused(status, "df_fp8_gemm_blocks", gemm(**kw))


def norm(q=True, dtype=F32, x=FAKE, rows=4, cols=8, ldx=8, res=None, ldr=0, sum=None, lds=0, gamma=FAKE, eps=1e-5, y=FAKE + 64,
         ldy=8, rstd=None, fmt=0, codes=FAKE, ldq=16, kind=E8, scales=FAKE, ldsc=16):
    L = df.lib()
    if not q:
        return L.df_rmsnorm_forward(dtype, x, rows, cols, ldx, res, ldr, sum, lds, gamma, eps, y, ldy, rstd, None)
    return L.df_rmsnorm_quantize(dtype, x, rows, cols, ldx, res, ldr, sum, lds, gamma, eps, y, ldy, rstd, fmt, codes, ldq, kind,
                                 scales, ldsc, None)


@pytest.mark.parametrize("q", [False, True])
@pytest.mark.parametrize("status,kw", [
    (-1, dict(rows=-1)), (-1, dict(cols=-1)), (-2, dict(dtype=I8)), (-1, dict(eps=-1.0)), (-1, dict(eps=float("nan"))),
    (-1, dict(sum=FAKE + 128)), (-1, dict(x=None)), (-1, dict(ldx=7)), (-1, dict(ldy=7)), (-1, dict(res=FAKE, ldr=7)),
    (-1, dict(res=FAKE, ldr=8, sum=FAKE + 64, lds=8)), (-1, dict(res=FAKE, ldr=8, sum=FAKE + 128, lds=7)),
    (-1, dict(res=FAKE + 256, ldr=8, sum=FAKE, lds=9)), (-1, dict(y=FAKE, ldy=9)), (-4, dict(x=FAKE + 2)),
    (-4, dict(gamma=FAKE + 1)), (-4, dict(rstd=FAKE + 2)), (-1, dict(rows=0x7FFFFFFF)), (0, dict(rows=0, x=None)),
    (0, dict(cols=0, ldx=0, ldy=0)),
])
def test_norm_refusals(status, kw, q):
    refused(status, "df_rmsnorm", norm(q, **kw))


@pytest.mark.parametrize("status,kw", [
    (-1, dict(fmt=2)), (-1, dict(kind=2)), (-1, dict(codes=None)), (-1, dict(scales=None)), (-4, dict(ldq=8)),
    (-4, dict(codes=FAKE + 8)), (-4, dict(ldsc=8)), (-4, dict(rows=20, ldsc=16)), (-4, dict(scales=FAKE + 2)),
    (-4, dict(kind=SF, ldsc=5)),
])
def test_norm_codes_refusals(status, kw):
    refused(status, "df_rmsnorm_quantize", norm(**kw))


def test_norm_needs_y():
    refused(-1, "df_rmsnorm_forward", norm(False, y=None))


def bwd(dtype=F32, dy=FAKE, lddy=8, x=FAKE, ldx=8, rows=4, cols=8, gamma=FAKE, rstd=FAKE, eps=1e-5, dr=None, lddr=0, dx=FAKE,
        lddx=8, dg=FAKE, ws=FAKE, wsb=1 << 20):
    return df.lib().df_rmsnorm_backward(dtype, dy, lddy, x, ldx, rows, cols, gamma, rstd, eps, dr, lddr, dx, lddx, dg, ws, wsb,
                                        None)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(rows=-1)), (-1, dict(cols=-1)), (-2, dict(dtype=I8)), (-1, dict(eps=-1.0)), (-1, dict(dy=None)),
    (-1, dict(x=None)), (-1, dict(dx=None)), (-1, dict(lddy=7)), (-1, dict(ldx=7)), (-1, dict(lddx=7)),
    (-1, dict(dr=FAKE, lddr=7)), (-1, dict(lddx=9)), (-4, dict(dy=FAKE + 2)), (-4, dict(dg=FAKE + 1)),
    (-4, dict(rstd=FAKE + 2)), (-5, dict(ws=None)), (-5, dict(ws=FAKE + 8)), (-5, dict(wsb=4 * 8 * 4 + 15)),
    (0, dict(cols=0, dy=None, x=None, dx=None, ws=None, wsb=0)),
])
def test_norm_backward_refusals(status, kw):
    refused(status, "df_rmsnorm_backward", bwd(**kw))


def test_workspace_sizes():
    need = df.lib().df_rmsnorm_backward_workspace_bytes
    assert need(0, 5) == need(5, 0) == need(-1, 5) == 0
    assert need(4, 8) == 4 * 8 * 4 + 4 * 4 and need(16384, 1600) == 512 * 1600 * 4 + 16384 * 4
    moe_ws = df.lib().df_moe_layer_workspace_bytes
    for bad in ((0, 8, 8, 4, 2), (65, 8, 8, 4, 2), (1, 8, 8, 4, 17), (1, 8, 8, 4, 5), (1, 8, 0, 4, 2), (1, 0, 8, 4, 2),
                (1, 8, 8, 257, 2), (1, 8, 8, 4, 0)):
        assert moe_ws(*bad) == 0
    assert moe_ws(2, 8, 8, 4, 2) > 2 * 2 * 256 * 4


def moe(dtype=BF, x=FAKE, ldx=24, tokens=3, H=24, N=20, experts=6, top=2, ldt=F32, logits=FAKE, ldl=6, renorm=1, act=0, w1=FAKE,
        ldw1=32, w2=FAKE, ldw2=32, kind=E8, s1=FAKE, lds1=48, s2=FAKE, lds2=32, y=FAKE, ldy=24, ids=FAKE, wt=FAKE, ws=FAKE,
        wsb=1 << 20):
    return df.lib().df_moe_layer(dtype, x, ldx, tokens, H, N, experts, top, ldt, logits, ldl, renorm, act, w1, ldw1, w2, ldw2,
                                 kind, s1, lds1, s2, lds2, y, ldy, ids, wt, ws, wsb, None)


@pytest.mark.parametrize("status,kw", [
    (-2, dict(dtype=F32)), (-2, dict(ldt=I8)), (-1, dict(tokens=-1)), (-1, dict(H=-1)), (-1, dict(N=0)), (-1, dict(experts=0)),
    (-2, dict(tokens=65)), (-2, dict(experts=257, ldl=257)), (-1, dict(top=0)), (-1, dict(top=7)),
    (-1, dict(top=17, experts=20, ldl=20)), (-1, dict(act=3)), (-1, dict(kind=2)), (-1, dict(x=None)), (-1, dict(logits=None)),
    (-1, dict(w1=None)), (-1, dict(w2=None)), (-1, dict(s1=None)), (-1, dict(s2=None)), (-1, dict(y=None)),
    (-1, dict(ids=None)), (-1, dict(wt=None)), (-1, dict(ldx=23)), (-1, dict(ldy=23)), (-1, dict(ldl=5)),
    (-4, dict(x=FAKE + 1)), (-4, dict(logits=FAKE + 2)), (-4, dict(ids=FAKE + 2)), (-4, dict(ldw1=24)), (-4, dict(ldw2=16)),
    (-4, dict(w1=FAKE + 8)), (-4, dict(lds1=32)), (-4, dict(lds2=16)), (-4, dict(s1=FAKE + 4)), (-4, dict(kind=SF, lds2=26)),
    (-2, dict(N=1 << 20, ldw2=1 << 20, lds1=1 << 21, wsb=1 << 40, H=4096, ldx=4096, ldy=4096, ldw1=4096, lds2=4096)),
    (-5, dict(ws=None)), (-5, dict(ws=FAKE + 8)), (-5, dict(wsb=100)), (0, dict(tokens=0)), (0, dict(H=0)),
])
def test_moe_refusals(status, kw):
    refused(status, "df_moe_layer", moe(**kw))


def test_python_refusals():
    x = torch.zeros(4, 40)
    e8 = torch.float8_e8m0fnu
    codes = torch.zeros(4, 48, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.zeros(1, 16, dtype=torch.uint8).view(e8)[:, :4]
    for bad in (lambda: df.quantize_blocks(x), lambda: df.quantize_blocks(x[0]), lambda: df.quantize_blocks(x, want_q=False),
                lambda: df.gemm_blocks(codes, scales, codes, scales, 40),
                lambda: df.gemm_blocks(codes, scales, codes, scales, 49), lambda: df.gemm_blocks(codes, scales, codes, scales, -1),
                lambda: df.gemm_blocks(codes, scales[:, :3], codes, scales, 40),
                lambda: df.gemm_blocks(codes, scales.float(), codes, scales, 40),
                lambda: df.gemm_blocks(codes[:, 1:41], scales, codes, scales, 40),
                lambda: df.gemm_blocks(x, scales, codes, scales, 40), lambda: df.block_scales(torch.ones(3, 4), rows=400),
                lambda: df.block_scales(torch.ones(3)), lambda: df.rmsnorm_forward(x), lambda: df.rmsnorm_forward(x[0]),
                lambda: df.rmsnorm_quantize(x), lambda: df.rmsnorm_backward(x, x), lambda: df.rmsnorm_backward(x, x[0]),
                lambda: df.quantize_experts_blocks(x), lambda: df.quantize_experts_blocks(x[None])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        df.quantize_blocks(x, scale_dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        df.block_scales(torch.ones(3, 4, dtype=torch.int32))
    t = torch.zeros(2, 32, dtype=torch.bfloat16)
    w1 = torch.zeros(4, 32, 32, dtype=torch.uint8).view(torch.float8_e4m3fn)
    w2 = torch.zeros(4, 32, 16, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(4, 1, 32, dtype=torch.uint8).view(e8)
    logits = torch.zeros(2, 4)
    for bad in (lambda: df.moe_layer(t, logits, w1, s, w2, s, 0), lambda: df.moe_layer(t, logits, w1, s, w2, s, 5),
                lambda: df.moe_layer(t, logits, w1, s, w2, s, 2), lambda: df.moe_layer(t, logits[0], w1, s, w2, s, 2),
                lambda: df.moe_layer(t, logits, w1, s, w2, s, 2, activation="relu"),
                lambda: df.moe_layer(t, logits[:, :3], w1, s, w2, s, 2), lambda: df.moe_layer(t, logits, w1[:, :30], s, w2, s, 2),
                lambda: df.moe_layer(t, logits, w1, s, w2, s.float(), 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        df.moe_layer(t.float(), logits, w1, s, w2, s, 2)


def test_block_scales_on_the_cpu():
    s = torch.arange(15, dtype=torch.float32).view(5, 3)
    got = df.block_scales(s)
    assert torch.equal(got, s.t()) and got.stride(0) == 8
    got = df.block_scales(s[:2], rows=200)
    assert got.shape == (3, 200) and torch.equal(got[:, 127], s[0]) and torch.equal(got[:, 128], s[1])


@pytest.mark.parametrize("kw", [dict(M=2**31 - 1, N=1), dict(M=1, N=2**31 - 5), dict(M=2**31 - 1, N=2**31 - 1),
                                dict(M=2**28 + 1, N=3)])
@pytest.mark.parametrize("K", [0, 40])
def test_outputs_of_too_many_tiles(kw, K):
    """Sizes next to 2^31 are not lost in the count of tiles."""
    refused(-2, "df_fp8_gemm_blocks", gemm(K=K, ldsa=2**31 - 16, ldsb=2**31 - 16, ldc=2**31 - 1, **kw))
