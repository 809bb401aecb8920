"""cab_paged_attn_fwd: which scales it takes, without a GPU."""

import pytest

from cab_attention import _native as nat
from test_host_paged import FAKE, arr, lib


@pytest.mark.parametrize("scale", [0.0, 2.4e38, 3.4e38])
def test_scales_that_are_refused(lib, scale):
    """Also those whose product with log2(e) is past fp32: the largest score's weight would be 2^(0 inf)."""
    qs, pool = arr(8 * 128, 128, 128, 1), arr(2 * 16 * 128, 16 * 128, 128, 1)
    st = lib.cab_paged_attn_fwd(
        FAKE, FAKE + (1 << 32), FAKE + (1 << 33), nat.CAB_BF16, 3, 8, 2, 128, 900, 16, qs, pool, pool, qs, FAKE,
        500, 500, FAKE, scale, FAKE + (1 << 20), None, FAKE, 1 << 40, None)
    assert st == nat.CAB_EINVAL and b"scale" in lib.cab_last_error()
