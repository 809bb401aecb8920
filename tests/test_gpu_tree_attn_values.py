"""tree_attention on values that have no softmax, against the float64 oracle: which outputs
and log-sum-exps are NaN, which -inf, and that all others stay what they are."""

import numpy as np
import pytest
import torch

from oracle import spec_oracle as S
from test_gpu_tree_attn import ATOL, DT, LSE_ATOL, np64, rand

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def run(cuda, q, k, v, parents, n):
    from cab_attention.kernels import tree_attention
    out, lse = tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor(parents).int().to(cuda),
                              torch.tensor(n, dtype=torch.int32).to(cuda), return_lse=True)
    return np64(out), np64(lse)


def alike(got, want, dt):
    """NaN and infinities in the same places, finite values as near as finite inputs' (the
    tolerances of the plain cases: no score that is finite changes)."""
    for x, w, atol in zip(got, want, (ATOL[dt], LSE_ATOL)):
        assert np.array_equal(np.isnan(x), np.isnan(w))
        assert np.array_equal(np.isneginf(x), np.isneginf(w))
        assert np.array_equal(np.isposinf(x), np.isposinf(w))
        ok = np.isfinite(w)
        np.testing.assert_allclose(x[ok], w[ok], atol=atol, rtol=0)


# One K / V head and as many query heads: 4, 20 rows (rows_kernel, fp32 at 20 with the second
# tile of rows), 60, 120 and 180 rows (the tiles of 64, 128 and 256).
ROWS = [(1, 4), (2, 10), (6, 10), (6, 20), (9, 20)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("H,T", ROWS)
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("where", ["context", "last", "draft", "query"])
def test_bad_scores(cuda, dt, H, T, bad, where):
    """A bad value in a key of the context (an early one, and the last, whose tile is not
    full), in a draft's key or in one node's query: each row that sees it has the oracle's
    NaN, or, where its score is -inf, a softmax without that key."""
    B, N, D = 2, 700, 64
    n = [601, 130]
    q, k, v = rand((B, H, T, D), dt, 1), rand((B, 1, N, D), dt, 2), rand((B, 1, N, D), dt, 3)
    parents = np.array([[-1] + [(i - 1) // 2 for i in range(1, T)]] * B)
    parents[1, T - 1] = -2
    if where == "context":
        k[0, 0, 70, 5] = bad
    elif where == "last":
        k[0, 0, n[0] - 1, 5] = bad
    elif where == "draft":
        k[0, 0, n[0] + 1, 5] = bad
    else:
        q[0, H - 1, 1, 5] = bad
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, n)
    # (the test itself: the other sequence is finite but for its absent node)
    assert np.isnan(want[1][0]).any() or np.isinf(bad)
    assert np.isfinite(want[1][1, :, :T - 1]).all()
    assert np.isneginf(want[1]).sum() == H
    alike(run(cuda, q, k, v, parents, n), want, dt)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("H,T", ROWS)
@pytest.mark.parametrize("length", [0, 33, 300])
def test_all_scores_minus_infinity(cuda, dt, H, T, length):
    """Nodes whose every score is -inf have no softmax (NaN), unlike absent ones (0, -inf)."""
    B, N, D = 1, 400, 64
    q, k, v = rand((B, H, T, D), dt, 1), rand((B, 1, N, D), dt, 2), rand((B, 1, N, D), dt, 3)
    k[..., 0] = k[..., 0].abs() + 1
    q[:, :, 1, 0] = -INF
    parents = np.array([[-1] + [0] * (T - 2) + [T]])
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, [length])
    assert np.isnan(want[1][:, :, 1]).all() and np.isneginf(want[1][:, :, T - 1]).all()
    assert np.isfinite(want[1][:, :, 2:T - 1]).all()
    alike(run(cuda, q, k, v, parents, [length]), want, dt)


def test_totals_of_a_commit(cuda):
    """Importance totals fed by such a log-sum-exp are NaN, as update()'s weights would make
    them, not infinite."""
    from cab_attention.kernels import key_scores, tree_attention
    q, k = torch.randn((1, 2, 3, 64), device=cuda), torch.randn((1, 2, 40, 64), device=cuda)
    q[0, 0, 1, 3] = NAN
    up = torch.tensor([-1, 0, 1], dtype=torch.int32, device=cuda)
    _, lse = tree_attention(q, k, k, up, return_lse=True)
    totals = key_scores(q, k, lse, causal=True)
    assert not torch.isinf(totals).any() and torch.isnan(totals[0, 0, :39]).all()
    assert torch.isfinite(totals[0, 1]).all()
