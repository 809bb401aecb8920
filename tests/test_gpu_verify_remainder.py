"""verify_drafts after rejected tokens that held nearly all of a row's weight: what is left
decides about their siblings, small as it is against the row's sum."""

import math

import numpy as np
import pytest
import torch

from oracle import spec_oracle as S
from test_gpu_verify import DT, MARGIN, check

pytestmark = pytest.mark.gpu


def row(V, weights, dt):
    """Logits of such weights, the rest masked."""
    x = torch.full((V,), -math.inf)
    for i, w in weights.items():
        x[i] = math.log(w)
    return x.to(DT[dt])


# Behind one token of weight 1, seven of 5e-8 (each below half a step of an fp32 sum of 1)
# beside it, and two siblings: 8e-7 and 5e-7 of the 1.65e-6 that are left.
SMALL = {i: 5e-8 for i in range(17, 24)}
ONE = {16: 1.0, **SMALL, 2000: 8e-7, 3000: 5e-7}
# Two tokens of about half each first.
TWO = {16: 1.0, 1024: 0.9, **SMALL, 2000: 8e-7, 3000: 5e-7}


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("V", [4096, 50001])
@pytest.mark.parametrize("r1,r2", [(0.51, 0.5), (0.55, 0.5), (0.55, 0.62), (0.45, 0.3), (0.6, 0.99)])
@pytest.mark.parametrize("weights,big", [(ONE, [16]), (TWO, [16, 1024]), (TWO, [1024, 16])])
def test_siblings_of_nearly_all_weight(cuda, dt, V, r1, r2, weights, big):
    n = len(big)
    tokens = [0, *big, 2000, 3000]
    T = len(tokens)
    parents = torch.tensor([-1] + [0] * (T - 1), dtype=torch.int32)
    logits = torch.stack([row(V, weights, dt)] * T)[None]
    # The large ones' uniform numbers reject them: the largest fp32 below 1 for the last of them.
    u = [0.0] + [0.9] * (n - 1) + [1 - 2.0 ** -24, r1, r2]
    rng = np.random.default_rng(V)
    noise = torch.from_numpy(rng.exponential(size=(1, V)).astype(np.float32))
    x = dict(logits=logits, drafts=None, tokens=torch.tensor([tokens]), parents=parents,
             uniforms=torch.tensor([u], dtype=torch.float32), noise=noise, temperature=1.0)
    assert check(x, cuda, MARGIN)[0] in (1, 2)


def test_long_rows(cuda):
    """The same where rows are read by the walk itself (logits past 2^28 bytes), with a
    rejected child at every node of a chain of such rows, and a row summed anew twice."""
    from cab_attention.kernels import verify_drafts
    V = 9_000_000
    steps = {16: 1.0, **SMALL, 2000: 1e-3, 3000: 8e-7, 4000: 5e-7, V - 1: 1e-7}
    tokens = [0, 16, 2000, 3000, 4000, 16, 2000, 3000]
    parents = torch.tensor([-1, 0, 0, 0, 0, 4, 4, 4], dtype=torch.int32)
    for r3, r4, r7 in ((0.46, 0.5, 0.46), (0.36, 0.9, 0.4), (0.56, 0.45, 0.2)):
        logits = torch.stack([row(V, steps, "fp32")] * 8)[None]
        u = torch.tensor([[0.0, 1 - 2.0 ** -13, 0.9995, r3, r4, 1 - 2.0 ** -13, 0.9995, r7]])
        noise = torch.from_numpy(np.random.default_rng(3).exponential(size=(1, V)).astype(np.float32))
        path, token, m = S.verify(logits[0].numpy(), tokens, parents.tolist(), u[0].numpy(), noise[0].numpy(), 1.0)
        assert m > MARGIN
        got = verify_drafts(logits.to(cuda), torch.tensor([tokens], device=cuda), parents.to(cuda),
                            u.to(cuda), noise.to(cuda), 1.0)
        assert got[0][0].tolist() == path + [-1] * (8 - len(path))
        assert int(got[1]) == len(path) and int(got[2]) == token
