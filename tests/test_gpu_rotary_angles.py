"""The sines and cosines of Rotary by themselves: pairs (1, 0) and (0, 1) turn into them."""

import numpy as np
import pytest
import torch

from cab_attention.kernels import Rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
def test_sines_and_cosines(cuda, interleaved):
    """At positions of every size. The angle is formed modulo a turn to 2 pi (2^-33 + 2^31 2^-65), which is
    1.5e-9; what is left of it after the nearest quarter turn, up to pi / 4, is rounded three times (to 24
    bits, its factor, their product): 3 pi / 4 2^-24. The polynomials add 1.9e-9 and five roundings of 2^-24 of terms
    that fall fast from 1: two of them at the most. The products with 1 and 0 are exact."""
    rot = Rotary(128, interleaved=interleaved).to(cuda)
    rng = np.random.default_rng(0)
    at = np.concatenate((np.arange(4000), rng.integers(0, 1 << 20, 20000), rng.integers(-(1 << 31), 1 << 31, 20000)))
    x = torch.zeros((1, 2, len(at), 128), device=cuda)
    first, second = ((slice(0, 128, 2), slice(1, 128, 2)) if interleaved else (slice(0, 64), slice(64, 128)))
    x[0, 0, :, first], x[0, 1, :, second] = 1.0, 1.0
    got = rot(x, positions=torch.tensor(at, dtype=torch.int32, device=cuda)).double().cpu().numpy()
    # The oracle's angle, exactly: whole numbers of 2^-64 turns, modulo 2^64.
    turns = (at.astype(object)[:, None] * np.array([int(t) for t in rot.turns.tolist()], dtype=object)) % (1 << 64)
    angle = (turns >> 11).astype(np.float64) * 2.0 ** -53 * 2 * np.pi
    bound = 3 * np.pi / 4 * 2.0 ** -24 + 2 * 2.0 ** -24 + 1.5e-9 + 1.9e-9
    for y, want in ((got[0, 0, :, first], np.cos(angle)), (got[0, 0, :, second], np.sin(angle)),
                    (got[0, 1, :, first], -np.sin(angle)), (got[0, 1, :, second], np.cos(angle))):
        assert np.abs(y - want).max() <= bound
