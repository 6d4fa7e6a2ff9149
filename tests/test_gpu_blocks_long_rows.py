"""A row of more than 4 GiB through the quantizer: the codes and scales of its far columns
are those of the same columns as a row of their own."""
import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tail", [1, 300, 384])
def test_far_columns(dev, tail):
    start, rows = 2 ** 30, 2  # 2^32 bytes of fp32
    g = torch.Generator(device=dev).manual_seed(tail)
    x = torch.ones(rows, start + tail, device=dev)
    x[:, :128] = torch.randn(rows, 128, generator=g, device=dev) * 3
    x[:, start - 128:] = torch.randn(rows, 128 + tail, generator=g, device=dev)
    near = x[:, start - 128:].contiguous()
    raw = lambda t: t.contiguous().view(torch.uint8)
    q, s, _, _ = df.quantize_blocks(x)
    nq, ns, _, _ = df.quantize_blocks(near)
    assert torch.equal(raw(q[:, start - 128:]), raw(nq)) and torch.equal(raw(s[start // 128 - 1:]), raw(ns))
    del q, s
    _, _, qt, st = df.quantize_blocks(x, want_q=False, want_qt=True)
    _, _, nqt, nst = df.quantize_blocks(near, want_q=False, want_qt=True)
    assert torch.equal(raw(qt[start - 128:]), raw(nqt)) and torch.equal(raw(st[:, start - 128:]), raw(nst))
