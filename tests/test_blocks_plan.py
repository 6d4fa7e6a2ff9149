"""Refusals of df_fp8_gemm_blocks_plan (CPU only)."""
import ctypes

import pytest

import deepfuse_amd as df
from deepfuse_amd import DType

F32, BF, I8 = (int(d) for d in (DType.FLOAT32, DType.BFLOAT16, DType.INT8))


@pytest.mark.parametrize("status,args", [
    (-1, (0, 5, 40, 1, BF)), (-1, (5, 0, 40, 1, BF)), (-1, (5, 5, -1, 1, BF)), (-1, (5, 5, 40, 2, BF)), (-2, (5, 5, 40, 1, I8)),
    (-2, (1 << 18, 1 << 18, 40, 1, BF)), (0, (5, 5, 0, 0, F32)), (0, (5, 5, 2**31 - 1, 1, BF))])
def test_refusals(status, args):
    k = ctypes.c_int(-7)
    assert df.lib().df_fp8_gemm_blocks_plan(*args, ctypes.byref(k)) == status
    assert (k.value == -7) == (status != 0)
    if status:
        assert "df_fp8_gemm_blocks_plan" in df.lib().df_last_error_string().decode()


def test_no_output():
    assert df.lib().df_fp8_gemm_blocks_plan(5, 5, 40, 1, BF, None) == -1
