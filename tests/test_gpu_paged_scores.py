"""paged_attention: scores of any finite size."""

import math

import numpy as np
import pytest
import torch

from cab_attention.kernels import paged_attention
from test_gpu_paged_attn import ATOL, DT, np64, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("size", [1e8, 1e12, 1e20, 1e31, 1e36])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_of_any_finite_size(cuda, dt, n, size, sign):
    """Scores around +-size: the largest one's V row, or the mean of all where they are equal; and with a scale that
    brings them to usual sizes, the softmax."""
    host, (q, k, v, table, m) = setup(1, 2, 1, 64, 16, [n], dt, cuda)
    q.zero_()
    q[..., 0] = math.sqrt(size)
    k[..., 0] = sign * math.sqrt(size)
    see = lambda: (np64(x) for x in paged_attention(q, k, v, table, m, return_lse=True))
    score = float(q[0, 0, 0, 0]) * float(k[0, 0, 0, 0])
    rows = v[table[0].long(), 0].reshape(-1, 64)[:n]
    out, lse = see()
    np.testing.assert_allclose(out[0, 0, 0], np64(rows).mean(0), atol=ATOL[dt], rtol=0)
    np.testing.assert_allclose(lse, score / 8 + math.log(n), rtol=2.0 ** -21)
    for key in (0, 17, n - 1):
        k[..., 0] = sign * math.sqrt(size)
        k[int(table[0, key // 16]), 0, key % 16, 0] *= 2.0 if sign > 0 else 0.5
        out, lse = see()
        assert np.array_equal(out[0, 0, 0], np64(rows[key]))
        np.testing.assert_allclose(lse, score / 8 * (2.0 if sign > 0 else 0.5), rtol=2.0 ** -21)
    # Scores of up to 8 with their sign, once scaled.
    x = torch.linspace(0.25, 1.0, n, dtype=torch.float64).to(DT[dt]) * (sign * math.sqrt(size))
    pad = torch.zeros(len(table[0]) * 16, dtype=DT[dt])
    pad[:n] = x
    k[table[0].long(), 0, :, 0] = pad.view(-1, 16).to(cuda)
    scale = 8.0 / size
    out, lse = (np64(y) for y in paged_attention(q, k, v, table, m, scale=scale, return_lse=True))
    z = np64(q)[0, 0, 0, 0] * np64(pad[:n]) * float(np.float32(scale))
    w = np.exp(z - z.max())
    np.testing.assert_allclose(lse, z.max() + math.log(w.sum()), atol=2e-5, rtol=0)
    np.testing.assert_allclose(out[0, 0, 0], w / w.sum() @ np64(rows), atol=ATOL[dt], rtol=0)
