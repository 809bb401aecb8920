"""adjust_logits: what the repetition penalty makes of a value in 16 bits."""

import numpy as np
import pytest
import torch

from cab_attention.kernels import adjust_logits

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("r", [0.6, 1.1, 1.2, 1.3, 2.4, 3.6])
@pytest.mark.parametrize("biases", [0, 1])
def test_quotients_are_the_fp32_ones(cuda, dt, r, biases):
    """Every positive value over r is the fp32 quotient, rounded to the type. At 6 / 5 and its like a twelfth
    of the exact quotients lie so near the border of two 16-bit values that a product with a rounded 1 / r falls on
    the other side. (Values from 2^-100 up: below them the remainder of a quotient is no normal number.)"""
    x = torch.arange(1, 0x7f80 if dt == "bf16" else 0x7c00, dtype=torch.int16).view(DT[dt])
    x = x[x.float() >= 2.0 ** -100]
    r = float(np.float32(r))
    n = len(x)
    got = adjust_logits(x.to(cuda)[None, None], torch.arange(n, device=cuda)[None], repetition=r,
                        prompt_lengths=torch.tensor([n], device=cuda),
                        bias_tokens=torch.full((1, biases), n, device=cuda) if biases else None,
                        bias=torch.ones((1, biases), device=cuda) if biases else None)[0, 0].cpu()
    assert torch.equal(got, (x.double() / r).float().to(DT[dt]))
