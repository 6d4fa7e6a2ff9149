"""df_moe_layer where experts take many tokens, so that an expert's are several units of
W2 and blocks share its columns: against the definition in binary64, by the bars of
test_gpu_moe.py, the same bits each time, and in a captured graph."""
import pytest
import torch

import deepfuse_amd as df
from test_gpu_moe import E8, check, make

pytestmark = pytest.mark.gpu

# tokens, experts, top, H, N
DENSE = [(64, 8, 8, 400, 1600), (64, 4, 4, 768, 1024), (32, 4, 2, 771, 3000), (64, 2, 2, 130, 1030), (64, 16, 16, 320, 400),
         (33, 3, 3, 515, 771), (64, 1, 1, 64, 4100)]


@pytest.mark.parametrize("act", ["swiglu", "gelu"])
@pytest.mark.parametrize("kind", [E8, torch.float32])
@pytest.mark.parametrize("T,E,top,H,N", DENSE)
def test_dense(dev, T, E, top, H, N, kind, act):
    t = make(dev, T, E, H, N, act, torch.bfloat16, kind)
    first = df.moe_layer(*t, top, activation=act)
    check(first, *t, top, act)
    assert all(torch.equal(a, b) for a, b in zip(df.moe_layer(*t, top, activation=act), first))


def test_skewed(dev):
    """All tokens' first choice is one expert, the others' units are few."""
    x, logits, *w = make(dev, 64, 8, 400, 1600)
    logits[:, 5] += 100
    check(df.moe_layer(x, logits, *w, 4), x, logits, *w, 4, "swiglu")


def test_dense_captured(dev):
    t, u = make(dev, 64, 8, 400, 1600), make(dev, 64, 8, 400, 1600, seed=1)
    want = [df.moe_layer(*v, 8) for v in (t, u)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = df.moe_layer(*t, 8)
    x = t[0].clone()
    for i in range(4):
        t[0].copy_(x)
        graph.replay()
        eager = df.moe_layer(*u, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0])) and all(torch.equal(a, b) for a, b in zip(eager, want[1]))


def test_workspace_grows_with_the_units(dev):
    """As many shares as the units' steps ask for, not an expert's one: their sums' room."""
    need = df.lib().df_moe_layer_workspace_bytes
    assert need(64, 1600, 1600, 8, 8) - need(64, 1600, 1, 8, 8) > 2 * 64 * 8 * (1792 - 256) * 2 + 5 * 64 * 1600 * 4 - 1
    assert need(64, 1600, 400, 16, 4) - need(64, 1600, 1, 16, 4) == 2 * 64 * 4 * 256 * 2
