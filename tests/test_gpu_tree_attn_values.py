"""tree_attention on values that have no softmax, against the float64 oracle: which outputs
and log-sum-exps are NaN, which -inf, and that all others stay what they are."""

import numpy as np
import pytest
import torch

from oracle import spec_oracle as S
from test_gpu_tree_attn import ATOL, DT, LSE_ATOL, np64, rand, trees

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


@pytest.mark.parametrize("dt,sink", [("fp16", 34.8125), ("bf16", 34.75)])
@pytest.mark.parametrize("H,T", [(1, 4), (2, 10), (4, 10), (5, 20), (10, 20)])
def test_small_weights_add_up(cuda, dt, sink, H, T):
    """One score 17.4 above 140000 others, whose V alone is not 0, in as many sequences as keep
    a context in one workgroup's stretch: a weight of 2.8e-8 each, together 0.4 % of the row. All
    weights are alike, so each result is n w / (1 + n w) for the n keys it sees; it is off by
    half a step of a weight's rounding and half a step of its own, and by fp32 sums: l's of 2188
    tiles onto 1 (2^-24 each, 1.4e-4), O's of twice as many products (2^-24 of it, 2.6e-4)."""
    B, N, D, length = 512, 140000 + T, 64, 140000
    from cab_attention.kernels import tree_attention
    k = torch.zeros((1, 1, N, D), dtype=DT[dt], device=cuda)
    v = torch.ones_like(k)
    k[0, 0, 0, 0], v[0, 0, 0] = sink, 0
    q = torch.zeros((B, H, T, D), dtype=DT[dt], device=cuda)
    q[..., 0] = 4
    parents = torch.arange(-1, T - 1, dtype=torch.int32, device=cuda)
    out, lse = tree_attention(q, k.expand(B, 1, N, D), v.expand(B, 1, N, D), parents, return_lse=True)
    w = np.exp(-4 * sink / 8)
    n = length - 1 + np.arange(1, T + 1)  # a chain: node i sees i + 1 drafts
    rel = torch.finfo(DT[dt]).eps
    want = np.broadcast_to((n * w / (1 + n * w))[:, None], (T, D))
    np.testing.assert_allclose(np64(out), np.broadcast_to(want, out.shape), rtol=rel + 4e-4, atol=0)
    np.testing.assert_allclose(np64(lse), np.broadcast_to(4 * sink / 8 + np.log1p(n * w), lse.shape),
                               atol=1.4e-4, rtol=0)


@pytest.mark.parametrize("H,T", ROWS)
@pytest.mark.parametrize("big", [1000, 9632, 9648, 9664, 30000])
def test_large_fp16_scores(cuda, H, T, big):
    """Scores of 1e5 to 1e8 in fp16, around the border past which weights are not scaled
    up: keys of a few scores that fp32 holds exactly, one or two maxima away from each other,
    the larger ones late. (The context's weights are all relative to one rounded level; a log-sum-exp
    has five roundings of the score's size.)"""
    from cab_attention.kernels import tree_attention
    N, D = 1000 + T, 64
    g = torch.Generator().manual_seed(T)
    q, k = torch.zeros((1, H, T, D)), torch.zeros((1, 1, N, D))
    q[..., 0], k[..., 0] = big, big
    step = 64.0 if big > 20000 else 8.0  # a multiple of the step of big^2 in fp32
    q[..., 1] = 1
    k[..., 1] = step * torch.randint(0, 3, (N,), generator=g)
    k[:, :, 700:1000, 1] += 8 * step  # (later, larger; the drafts weigh little)
    v = rand((1, 1, N, D), "fp16", 3)
    q, k = q.half(), k.half()
    parents = trees(1, T, "tree", T)
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, [1000])
    out, lse = tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor(parents).int().to(cuda),
                              torch.tensor([1000], dtype=torch.int32).to(cuda), return_lse=True)
    np.testing.assert_allclose(np64(out), want[0], atol=ATOL["fp16"], rtol=0)
    np.testing.assert_allclose(np64(lse), want[1], rtol=5 * 2 ** -24, atol=1e-5)


@pytest.mark.parametrize("H,T", ROWS)
@pytest.mark.parametrize("late", [True, False])
def test_fp16_scores_across_the_levels_border(cuda, H, T, late):
    """Scores of 2^24 / log2(e) less and more a few, the larger ones in the later keys or the
    earlier: sums taken on one side of the border are carried over to the other. (Each score is
    a whole number that fp32 sums exactly: 11629072 + 8 i + j.)"""
    N, D = 1300 + T, 64
    g = torch.Generator().manual_seed(T)
    q, k = torch.zeros((1, H, T, D)), torch.zeros((1, 1, N, D))
    q[..., :3] = torch.tensor([9640.0, 2.0, 8.0])
    k[..., 0] = 9640
    low = torch.tensor([51488.0, 5.0]) + torch.stack([torch.zeros(N), torch.randint(0, 3, (N,), generator=g)], 1)
    high = torch.tensor([51520.0, 0.0]) + torch.stack([torch.zeros(N), torch.randint(0, 2, (N,), generator=g)], 1)
    first = (torch.arange(N) < 650)[:, None]
    k[0, 0, :, 1:3] = torch.where(first == late, low, high)
    k[:, :, 1300:, 1] = 0  # (the drafts weigh nothing)
    v = rand((1, 1, N, D), "fp16", 3)
    q, k = q.half(), k.half()
    s = np64(k)[0, 0, :1300] @ np64(q)[0, 0, 0] / 8
    assert np.unique(s).tolist() == [11629077, 11629078, 11629079, 11629080, 11629081]
    parents = trees(1, T, "tree", T)
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, [1300])
    out, lse = run(cuda, q, k, v, parents, [1300])
    np.testing.assert_allclose(out, want[0], atol=ATOL["fp16"], rtol=0)
    np.testing.assert_allclose(lse, want[1], rtol=5 * 2 ** -24, atol=1e-5)
