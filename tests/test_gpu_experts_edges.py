"""dW next to rows whose codes are NaN, on every kernel that dW has: an expert's
tokens start and end at any byte of the transposed codes, and nothing of the
neighbours' bytes in its first and last 16 may reach it."""
import pytest
import torch

import deepfuse_amd as df

pytestmark = pytest.mark.gpu

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2

# tokens an expert: ranges that start and end off multiples of 16, both edges in one chunk of 16 (the 5, 1 and 3),
# an empty expert between others, whole chunks, and some steps of 128
COUNTS = [37, 21, 0, 70, 5, 1, 3, 150, 16, 209]

# outputs a tile wide or not: 3300 and more tiles of 32 x 32 go to large tiles; 256 x 128 ones for the first, whose
# units fit one round either way, 256 x 256 for the second (150 units against 300); small tiles for the third
FORMS = [(640, 1040, 5), (1040, 768, 10), (96, 100, 10)]


@pytest.mark.parametrize("N,K,E", FORMS, ids=["narrow", "wide", "small"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_neighbours_nan(dev, N, K, E, dt):
    counts = COUNTS[:E]
    b = [0]
    for c in counts:
        b.append(b[-1] + c)
    R = b[-1] + 9  # rows behind the last expert too
    ld = df.round16(R)
    g = torch.Generator(device=dev).manual_seed(N)
    a = torch.randint(-8, 9, (N, ld), generator=g, device=dev).float().to(E5)
    x = torch.randint(-8, 9, (K, ld), generator=g, device=dev).float().to(E4)
    off, s = torch.tensor(b, dtype=torch.int32, device=dev), torch.ones(1, device=dev)
    # whole numbers: exact in binary32 and in the fp8 instructions
    ref = torch.stack([a[:, lo:hi].float() @ x[:, lo:hi].float().t() for lo, hi in zip(b, b[1:])]).to(dt)
    for bad in [[e] for e in range(E) if counts[e]] + [[1, 3], list(range(0, E, 2)), list(range(1, E, 2))]:
        aq, xq = a.view(torch.uint8).clone(), x.view(torch.uint8).clone()
        for q in (aq, xq):
            q[:, b[-1]:] = 0x7F
            for e in bad:
                q[:, b[e]:b[e + 1]] = 0x7F
        got = df.experts_dw(aq, xq, off, R, s, s, out_dtype=dt)
        for e in range(E):
            if e in bad and counts[e]:
                assert got[e].isnan().all(), (bad, e)
            else:
                assert torch.equal(got[e], ref[e]), (bad, e)
