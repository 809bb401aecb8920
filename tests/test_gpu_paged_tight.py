"""paged_attention at every cut of test_gpu_paged_attn's cases, to the output's own rounding."""

import numpy as np
import pytest
import torch

from cab_attention.kernels import paged_attention
from oracle import paged_oracle as P
from test_gpu_paged_attn import CASES, DT, np64, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", CASES, ids=lambda c: str(c[:4]))
def test_only_the_output_is_rounded(cuda, case, dt, D):
    """Half a step of the output, and what fp32 makes of a mean of |v|: a score is a sum of D products, each
    sum off by 2^-24 of terms whose sizes add up to some 3 once scaled (400 * 2^-24 of its weight); a lane adds up
    its keys, one in 32 of a context (2^-24 each), and some 20 more join the lanes, waves and parts. Weights
    have 24 bits, in fp16 22."""
    B, H, Hkv, S, lengths = case
    host, args = setup(B, H, Hkv, D, S, lengths, dt, cuda, seed=1)
    q, k, v = (np64(x) for x in host[:3])
    out, _ = P.attention(q, k, v, host[3], lengths)
    mean, _ = P.attention(q, k, np.abs(v), host[3], lengths)
    keys = max(max(lengths), 0)
    off = np.abs(np64(paged_attention(*args)) - out)
    bound = (420 + keys / 32) * 2.0 ** -24 + (2.0 ** -22 if dt == "fp16" else 0.0)
    assert (off <= np.abs(out) * torch.finfo(DT[dt]).eps / 2 * (1 + 1e-6) + mean * bound + torch.finfo(DT[dt]).tiny).all()
