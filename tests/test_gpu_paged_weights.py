"""paged_attention: softmax weights in all their digits."""

import math

import numpy as np
import pytest
import torch

from cab_attention.kernels import paged_attention
from test_gpu_paged_attn import DT, np64

pytestmark = pytest.mark.gpu


def i32(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def plain_pages(keys, D, dt, cuda):
    """(K, V, table) of one sequence, whose pages of 16 are zeros in order."""
    pages = -(-keys // 16)
    k, v = (torch.zeros((pages, 1, 16, D), dtype=DT[dt], device=cuda) for _ in range(2))
    return k, v, torch.arange(pages, dtype=torch.int32, device=cuda)[None]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("columns", [2, 100])
def test_weights_keep_all_their_digits(cuda, dt, D, columns):
    """Two keys, V = 1 and -1, scores 0 and -t: tanh(t / 2), what is left of 1 - e^-t; in one workgroup, and in two parts.

    The scores are exact (one product that is not 0). The weight e^-t is off by its exponent's
    roundings, 2 t 2^-24, and the exponential's last place, at most 2^-23; the sums and quotient by 2^-23 of
    the result. With t up to 2^-4: below 2^-22 in all, halved by the sum of both weights, 2. Then the output's
    half step."""
    t = torch.tensor([2.0 ** -i * m for i in range(4, 15) for m in (1.0, 1.5, 1.8125)], dtype=torch.float64)
    q = torch.zeros((1, len(t), 1, D), dtype=DT[dt], device=cuda)
    q[0, :, 0, 3] = t.to(DT[dt]).to(cuda)
    k, v, table = plain_pages(16 * columns, D, dt, cuda)
    k[..., 3] = -math.inf  # (all other keys)
    k[0, 0, 5, 3], k[columns - 1, 0, 9, 3] = 0.0, -1.0
    v[0, 0, 5], v[columns - 1, 0, 9] = 1.0, -1.0
    out = np64(paged_attention(q, k, v, table, i32([16 * columns], cuda), scale=1.0))
    want = np.tanh(np64(q[..., 3]) / 2)[..., None]
    assert (np.abs(out - want) <= want * torch.finfo(DT[dt]).eps / 2 * (1 + 1e-6) + 2.0 ** -22).all()
