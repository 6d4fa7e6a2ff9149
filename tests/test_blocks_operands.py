"""Operands of codes that the products and the experts' layer read up to the next
multiple of 16 codes: what lies elsewhere, or nowhere, is refused (CPU only: the checks
come before a device is asked for)."""
import pytest
import torch

import deepfuse_amd as df
from deepfuse_amd import blocks

E8 = torch.float8_e8m0fnu


def codes(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def scales(blocks, rows):
    return df.block_scales(torch.ones(rows, blocks).to(E8))


def products_take(a):
    """Whether gemm_blocks takes these codes (and refuses the CPU behind them)."""
    K = a.shape[1]
    nb = -(-K // 128)
    with pytest.raises(ValueError) as e:
        df.gemm_blocks(a, scales(nb, a.shape[0]), codes(4, -(-K // 16) * 16), scales(nb, 4), K)
    assert "a_q" in str(e.value)
    with pytest.raises(ValueError) as f:
        df.gemm_blocks(codes(4, -(-K // 16) * 16), scales(nb, 4), a, scales(nb, a.shape[0]), K)
    took = ["16 bytes" not in str(x.value) for x in (e, f)]
    assert took[0] == took[1]
    return took[0]


def test_a_row_of_its_own_length():
    """One row that ends, with its storage or before other codes, at no multiple of 16."""
    assert not products_take(codes(1, 771))
    assert not products_take(codes(5, 771)[:1])  # (NaN codes of the row behind it would be its own)
    assert not products_take(codes(32, 771)[16:17])
    assert products_take(codes(1, 784)) and products_take(codes(1, 784)[:, :771])
    assert products_take(codes(5, 784)[2:3, :771]) and products_take(codes(5, 784)[4:, :771])
    assert products_take(codes(1, 16)[:, :1])


@pytest.mark.parametrize("rows", [1, 2, 7])
def test_storage_that_ends_inside_the_last_sixteen(rows):
    for size, ok in ((784 * rows, True), (784 * rows - 1, False), (784 * (rows - 1) + 771, False)):
        assert products_take(codes(size).as_strided((rows, 771), (784, 1))) is ok
    whole = codes(784 * rows)
    assert products_take(whole.as_strided((rows, 768), (784, 1), 16))


def layer_takes(w1, w2, H, N=40):
    """Whether moe_layer takes these weights, w1 [E, 2 N, >=H] and w2 [E, H, >=N]."""
    E = w1.shape[0]
    took = []
    for n, w, rows, cols in ((1, w1, 2 * N, H), (2, w2, H, N)):
        s = torch.ones(E, -(-cols // 128), -(-rows // 16) * 16).to(E8)[:, :, :rows]
        try:
            blocks._expert_weights("moe_layer", n, w, s, rows, cols, E)
            took.append(True)
        except ValueError as e:
            assert f"w{n} with strides" in str(e) and "16 bytes" in str(e)
            took.append(False)
    return took


def test_weights_that_end_inside_the_last_sixteen():
    H, N = 24, 40
    w1, w2 = codes(2, 2 * N, 32), codes(2, H, 48)
    assert layer_takes(w1, w2, H) == layer_takes(w1[:, :, :H], w2[:, :, :N], H) == [True, True]
    cut1 = codes(2 * 2 * N * 32 - 8).as_strided((2, 2 * N, H), (2 * N * 32, 32, 1))
    cut2 = codes(2 * H * 48 - 1).as_strided((2, H, N), (H * 48, 48, 1))
    assert layer_takes(cut1, cut2, H) == [False, False]
    # one expert with one row a matrix: its own stride decides
    w1 = codes(1, 2 * N, 16)[:, :, :1]
    assert layer_takes(w1, codes(1, 1, 48)[:, :, :N], 1) == [True, True]
    assert layer_takes(w1, codes(1, 1, N), 1) == [True, False]
    assert layer_takes(w1, codes(6, N)[None, 2:3], 1) == [True, False]


def test_no_columns():
    """The library writes nothing for H = 0, ids and weights neither."""
    x, logits = torch.zeros(2, 0, dtype=torch.bfloat16), torch.zeros(2, 4)
    w = codes(4, 32, 16), torch.zeros(4, 0, 32).to(E8), codes(4, 0, 16), torch.zeros(4, 1, 0).to(E8)
    with pytest.raises(ValueError, match="no columns"):
        df.moe_layer(x, logits, w[0], w[1], w[2], w[3], 2)


def test_operands_of_no_rows_and_no_codes():
    """As quantize_blocks and rmsnorm_quantize leave them for a batch of no tokens."""
    assert products_take(codes(0, 784)[:, :771])
    assert blocks._codes("f", "a_q", torch.empty(5, 0, dtype=torch.float8_e4m3fn), 0, True) == 0
    for nb in (0, 1, 3):
        for s in (torch.empty(nb, 0).to(E8), torch.empty(nb, 0), torch.empty(max(nb, 1), 0).as_strided((nb, 0), (0, 1))):
            assert blocks._scales_ld("f", "sa", s, nb, 0, s.dtype) == 0
