"""Every kernel of df_fp8_gemm_blocks, with each kind of scales and of outputs that can take
it, against binary64 by the bars of test_gpu_blocks_gemm.py.  Each size's kernel is asked
for and has to be the one meant: constants of the choice that move show here."""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import BlocksKernel as Kernel
from test_gpu_blocks_gemm import E4, E5, E8, check, operands

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
# sizes that every kind of call takes the same kernel for, and those that only some do
# (by scales, then whether the output is fp32); short, middling and long reductions
ALL = [(Kernel.T16, (1, 69, 3803)), (Kernel.T16, (71, 9, 553)), (Kernel.T16, (185, 1, 113)), (Kernel.T16X32, (13, 4201, 1613)),
       (Kernel.T16X32, (1, 7175, 45)), (Kernel.T16X32, (1, 7973, 525)), (Kernel.T32, (1851, 63, 307)), (Kernel.T32, (89, 2067, 75)),
       (Kernel.T32_LONG, (291, 857, 1859)), (Kernel.T32_LONG, (1079, 373, 1097)), (Kernel.T256X128, (7669, 2817, 161)),
       (Kernel.T256X128, (781, 5699, 839)), (Kernel.T256X128, (1919, 2979, 1345))]
SOME = {
    (E8, False): [(Kernel.T64, (1695, 363, 1881)), (Kernel.T64, (569, 1317, 645)), (Kernel.T128, (369, 3651, 69)),
                  (Kernel.T128, (6337, 135, 1055)), (Kernel.T128, (2753, 527, 4455)), (Kernel.T256, (4743, 5309, 211)),
                  (Kernel.T256, (6157, 1725, 303)), (Kernel.T256, (2045, 4595, 1107))],
    (E8, True): [(Kernel.T64, (1695, 363, 1881)), (Kernel.T64, (6057, 111, 515)), (Kernel.T64, (1961, 447, 299)),
                 (Kernel.T128, (923, 2193, 43)), (Kernel.T128, (5533, 355, 125)), (Kernel.T128, (1741, 1351, 985)),
                 (Kernel.T128, (4565, 629, 1229)), (Kernel.T256, (4743, 5309, 211)), (Kernel.T256, (6157, 1725, 303)),
                 (Kernel.T256, (2045, 4595, 1107))],
    (F32, False): [(Kernel.T64, (1695, 363, 1881)), (Kernel.T64, (569, 1317, 645)), (Kernel.T128, (369, 3651, 69)),
                   (Kernel.T128, (1741, 1351, 985)), (Kernel.T128, (2317, 767, 1367))],
    (F32, True): [(Kernel.T128, (369, 3651, 69)), (Kernel.T128, (1741, 1351, 985)), (Kernel.T128, (2317, 767, 1367))],
}
CASES = [(kind, out, k, s) for kind in (E8, F32) for out in (F32, BF, F16) for k, s in ALL + SOME[kind, out == F32]]


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind,out,kernel,size", CASES, ids=lambda v: str(v).replace("torch.", ""))
def test_kernel(dev, kind, out, kernel, size):
    M, N, K = size
    assert df.gemm_blocks_plan(M, N, K, kind, out) == kernel
    for fa in (E4, E5):
        a, sa, b, sb = operands(dev, M, N, K, fa, kind, seed=M)
        bias = torch.randn(N, device=dev) if fa == E4 else None
        check(df.gemm_blocks(a, sa, b, sb, K, bias=bias, out_dtype=out), a, sa, b, sb, K, bias)


def test_every_kernel_is_here():
    """What the choice offers: 256 x 256 tiles for powers of two, 64 x 64 for all but fp32
    scales with fp32 outputs."""
    for kind in (E8, F32):
        for out in (F32, BF, F16):
            want = set(Kernel) - ({Kernel.T256} if kind == F32 else set()) - ({Kernel.T64} if kind == out == F32 else set())
            assert {k for kd, o, k, _ in CASES if kd == kind and o == out} == want


def test_nothing_to_reduce(dev):
    assert df.gemm_blocks_plan(300, 290, 0) == Kernel.T32
