"""paged_attention: infinite values behind weights of any size."""

import math

import numpy as np
import pytest
import torch

from cab_attention.kernels import paged_attention
from test_gpu_paged_attn import DT, np64, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("low", [10.0, 20.0, 30.0, 60.0])
def test_infinite_values_behind_small_weights(cuda, dt, n, low):
    """One key's score lies `low` above all others, so that theirs weigh e^-low: infinities in their V rows are
    the output's, opposite ones NaN, and so is an infinity behind a score of -inf (0 times it). The other
    values are as without, to the least operands of their weights (in fp16 2^-38 of the largest, 3000 of them
    times values up to 5: 6e-8) and the output's step."""
    host, (q, k, v, table, m) = setup(1, 2, 1, 64, 16, [n], dt, cuda)
    q.zero_()
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[int(table[0, 1]), 0, 4, 0] = low  # (8 low / sqrt(64))
    dead = (int(table[0, (n - 1) // 16]), 0, (n - 1) % 16)
    k[(*dead, 0)] = -math.inf
    clean = np64(paged_attention(q, k, v, table, m))
    v2 = v.clone()
    inf = math.inf
    for key, d, x in ((3, 7, inf), (30, 9, -inf), (20, 12, inf), (5, 13, inf), (n - 3, 13, -inf), (n - 3, 20, inf)):
        v2[int(table[0, key // 16]), 0, key % 16, d] = x
    v2[(*dead, 30)] = inf
    out = np64(paged_attention(q, k, v2, table, m))[0, :, 0]
    assert (out[:, [7, 12, 20]] == inf).all() and (out[:, 9] == -inf).all() and np.isnan(out[:, [13, 30]]).all()
    rest = np.delete(np.arange(64), [7, 9, 12, 13, 20, 30])
    np.testing.assert_allclose(out[:, rest], clean[0, :, 0][:, rest], rtol=torch.finfo(DT[dt]).eps * 1.01, atol=1e-6)
