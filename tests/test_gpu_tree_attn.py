"""tree_attention against the float64 oracle, which picks each node's keys out one by one:
at the edges of the context's cuts (32-key steps, 64-key tiles), of the row tiles (16, 32,
64, 128, 256 rows a K / V head), of the trees (one node, chains, stars, absent nodes), and
with values that must not reach a row."""

import numpy as np
import pytest
import torch

from oracle import spec_oracle as S

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# Each weight's rounding to 16 bits moves an output, a mean of values of up to about 5, by
# at most half a step (bf16 2^-9 of the weight), and so does the output's own rounding (of a
# value up to about 4): together below 2 * 5 * 2^-9 (bf16), 2 * 5 * 2^-12 (fp16); fp32: sums of
# D + 256 terms, each off by 2^-24. The log-sum-exp is fp32 throughout: scores of up to
# about 8, their sums and the exponentials' errors, 2^-24 each.
ATOL = {"bf16": 2e-2, "fp16": 2.5e-3, "fp32": 2e-5}
LSE_ATOL = 2e-5


def trees(B, T, shape, seed):
    rng = np.random.default_rng(seed)
    out = np.full((B, T), -1)
    for b in range(B):
        for i in range(T):
            if shape == "chain":
                out[b, i] = i - 1
            elif shape == "star":
                out[b, i] = -1 if i == 0 else 0
            elif shape == "roots":
                out[b, i] = -1 if i % 3 == 0 else i - 1
            else:
                out[b, i] = -1 if i == 0 else int(i * rng.random())
    return out


def rand(shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(DT[dt])


def np64(t):
    return t.detach().double().cpu().numpy()


def close(out, lse, want, dt):
    w_out, w_lse = want
    gone = np.isneginf(w_lse)
    got = np64(lse)
    assert np.array_equal(np.isneginf(got), gone)
    np.testing.assert_allclose(got[~gone], w_lse[~gone], atol=LSE_ATOL, rtol=0)
    np.testing.assert_allclose(np64(out), w_out, atol=ATOL[dt], rtol=0)
    assert not np64(out)[gone].any()


CASES = [  # B, H, H_kv, T, N, lengths, shape
    (1, 4, 4, 1, 1, [0], "chain"),                  # the token alone
    (2, 8, 2, 1, 200, [31, 199], "chain"),          # 4 rows
    (3, 14, 2, 2, 300, [32, 33, 298], "chain"),     # 14 rows, 32-key steps' edges
    (2, 4, 1, 4, 600, [129, 128], "tree"),          # 16 rows, one step past four
    (2, 4, 4, 17, 700, [0, 640], "tree"),           # 17 rows: the second row tile
    (1, 8, 2, 8, 1500, [1492], "star"),             # 32 rows
    (2, 3, 1, 11, 900, [64, 63], "tree"),           # 33 rows: tiles, one full and one short
    (1, 4, 1, 16, 2000, [1089], "roots"),           # 64 rows
    (2, 5, 1, 13, 800, [1, 400], "tree"),           # 65 rows: 128-row tiles
    (1, 8, 2, 32, 1300, [1025], "tree"),            # 128 rows
    (1, 3, 1, 43, 500, [449], "tree"),              # 129 rows: 256-row tiles
    (1, 8, 2, 64, 1100, [1000], "tree"),            # 256 rows
    (2, 4, 2, 129, 700, [0, 571], "chain"),         # 258 rows: a second row tile
    (1, 2, 1, 256, 600, [65], "tree"),              # the most nodes
    (1, 2, 2, 256, 256, [0], "chain"),              # no room for a context
    (4, 2, 1, 3, 70, [-5, 67, 68, 2000], "chain"),  # lengths that count as 0, 67, 67, 67
]


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,H,Hkv,T,N,lengths,shape", CASES)
def test_against_oracle(cuda, B, H, Hkv, T, N, lengths, shape, dt, D):
    from cab_attention.kernels import tree_attention
    q = rand((B, T, H, D), dt, 1, 1.3).transpose(1, 2)
    k, v = rand((B, Hkv, N, D), dt, 2), rand((B, Hkv, N, D), dt, 3)
    parents = trees(B, T, shape, T)
    n = np.clip(lengths, 0, N - T)
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, n)
    for b in range(B):  # rows behind the drafts are not read
        k[b, :, n[b] + T:] = float("nan")
        v[b, :, n[b] + T:] = float("inf")
    out, lse = tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor(parents).int().to(cuda),
                              torch.tensor(lengths, dtype=torch.int32).to(cuda), return_lse=True)
    close(out, lse, want, dt)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("H,T", [(4, 7), (8, 20), (8, 40)])
def test_long_context_of_one_length(cuda, dt, H, T):
    """No lengths (the drafts are the last rows), one tree for all, many splits; K and V as
    a projection leaves them."""
    from cab_attention.kernels import tree_attention
    B, Hkv, N, D = 2, 2, 9001, 128
    q = rand((B, H, T, D), dt, 4, 1.3)
    k, v = (rand((B, N, Hkv, D), dt, s).transpose(1, 2) for s in (5, 6))
    parents = trees(1, T, "tree", T)
    want = S.tree_attention(np64(q), np64(k), np64(v), parents.repeat(B, 0), [N - T] * B, scale=0.07)
    out = torch.empty_like(q, device=cuda)
    got = tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor(parents[0]).to(cuda),
                         scale=0.07, out=out, return_lse=True)
    assert got[0] is out and out._version > 0
    close(*got, want, dt)


@pytest.mark.parametrize("dt,D,H,T,N", [("bf16", 128, 4, 35, 66200), ("fp16", 64, 5, 30, 66000),
                                        ("bf16", 64, 2, 16, 140000), ("fp16", 128, 1, 20, 140000)])
def test_long_lists(cuda, dt, D, H, T, N):
    """Lists past the sizes that send 129 to 256 rows to tiles of 128 and 17 to 32 to tiles: two
    heads of K and V and contexts of very unlike lengths."""
    from cab_attention.kernels import tree_attention
    B, Hkv = 2, 2
    q, k, v = rand((B, H * Hkv, T, D), dt, 1, 1.3), rand((B, Hkv, N, D), dt, 2), rand((B, Hkv, N, D), dt, 3)
    parents, n = trees(B, T, "tree", 4), [N - T, 700]
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, n)
    got = tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor(parents).to(cuda),
                         torch.tensor(n).to(cuda), return_lse=True)
    close(*got, want, dt)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("T", [6, 40])
def test_unseen_values_reach_nobody(cuda, dt, T):
    """Absent nodes, and siblings, full of NaN and infinities: only the rows that see them
    change, and absent rows are empty."""
    from cab_attention.kernels import tree_attention
    B, H, Hkv, N, D = 2, 4, 1, 300, 64
    q, k, v = rand((B, H, T, D), dt, 7), rand((B, Hkv, N, D), dt, 8), rand((B, Hkv, N, D), dt, 9)
    parents = trees(B, T, "tree", 12)
    parents[0, T - 2:] = -2                  # padding
    parents[1, 3] = 3                        # its own parent: no node, nor what hangs on it
    parents[1, 4] = 3
    parents[1, 5] = T + 7
    n = [100, 231]
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, n)
    gone = [[S.line(parents[b], i) is None for i in range(T)] for b in range(B)]
    for b in range(B):
        for i in range(T):
            if gone[b][i]:
                k[b, :, n[b] + i], v[b, :, n[b] + i] = float("nan"), float("inf")
                q[b, :, i] = float("nan")
    dev = [x.to(cuda) for x in (q, k, v)]
    up, lengths = torch.tensor(parents).to(cuda), torch.tensor(n).to(cuda)  # int64
    out, lse = tree_attention(*dev, up, lengths, return_lse=True)
    close(out, lse, want, dt)
    # A node that is there turns bad: its descendants and no others.
    dev[2][0, :, 100 + 1] = float("nan")
    bad, _ = tree_attention(*dev, up, lengths, return_lse=True)
    for i in range(T):
        line = S.line(parents[0], i)
        if line is not None and 1 in line:
            assert torch.isnan(bad[0, :, i]).all()
        else:
            assert torch.equal(bad[0, :, i], out[0, :, i])
    assert torch.equal(bad[1], out[1])


@pytest.mark.parametrize("dt", list(DT))
def test_large_scores(cuda, dt):
    """Scores of +-300 (one key takes the row), and a context all alike."""
    from cab_attention.kernels import tree_attention
    B, H, Hkv, T, N, D = 1, 4, 1, 9, 1000, 128
    q, k, v = rand((B, H, T, D), dt, 1, 30.0), rand((B, Hkv, N, D), dt, 2), rand((B, Hkv, N, D), dt, 3)
    k[:, :, 200:600] = k[:, :, 200:201]
    parents = trees(B, T, "tree", 5)
    w_out, w_lse = S.tree_attention(np64(q), np64(k), np64(v), parents, [900])
    out, lse = tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor(parents).to(cuda),
                              torch.tensor([900]).to(cuda), return_lse=True)
    # A score of 300 is off by up to (D + 2) 2^-24 of the sum of its terms' magnitudes (about
    # 2700 here), a weight by that factor: 2 * 0.021 * 5 in the worst case, about a 30th of it
    # as rounding errors add up.
    np.testing.assert_allclose(np64(lse), w_lse, atol=2e-3, rtol=0)
    np.testing.assert_allclose(np64(out), w_out, atol=ATOL[dt] + 7e-3, rtol=0)


@pytest.mark.parametrize("dt,H,T", [("bf16", 1, 1), ("bf16", 3, 7), ("fp32", 2, 2), ("fp16", 4, 40)])
@pytest.mark.parametrize("B,Hkv", [(70, 1), (131, 1), (17, 1), (33, 2)])
def test_many_sequences(cuda, B, Hkv, dt, H, T):
    """More sequences than a wave has lanes, more units than a quarter of the workgroups (whose
    stretches then run from one unit into the next), empty contexts among them."""
    from cab_attention.kernels import tree_attention
    N, D = 700 + T, 64
    rng = np.random.default_rng(B)
    n = np.where(rng.random(B) < 0.3, 0, rng.integers(0, 701, B))
    n[0], n[-1] = 0, 700
    q, k, v = rand((B, H * Hkv, T, D), dt, 1, 1.3), rand((B, Hkv, N, D), dt, 2), rand((B, Hkv, N, D), dt, 3)
    parents = trees(B, T, "tree", 2)
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, n)
    for b in range(B):
        v[b, :, n[b] + T:] = float("nan")
    got = tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor(parents).to(cuda),
                         torch.tensor(n).to(cuda), return_lse=True)
    close(*got, want, dt)


def test_far_rows(cuda):
    """A cache whose last sequence lies past 2^32 bytes, its context read at the end of it."""
    from cab_attention.kernels import tree_attention
    B, Hkv, N, D, T = 3, 1, 6_000_000, 128, 5
    big = torch.zeros((B, Hkv, N, D), dtype=torch.bfloat16, device=cuda)  # 4.6 GB
    big[2, :, -2000:] = rand((1, 2000, D), "bf16", 3).to(cuda)
    for H in (4, 16):
        q = rand((B, H, T, D), "bf16", 1)
        view = big[:, :, N - 2000:]
        parents = trees(B, T, "tree", 1)
        n = [0, 900, 1990]
        want = S.tree_attention(np64(q), np64(view), np64(view), parents, n)
        up, lengths = torch.tensor(parents).to(cuda), torch.tensor(n).to(cuda)
        close(*tree_attention(q.to(cuda), view, view, up, lengths, return_lse=True), want, "bf16")
        # The whole of a long row: its zeros weigh exp(0), the values at its end are in it.
        out, lse = tree_attention(q.to(cuda), big, big, up, None, return_lse=True)
        k = np64(big[2, 0, -2000:])
        s = np64(q)[2, 0, 0] @ k[:-T].T * D ** -0.5
        own = np64(q)[2, 0, 0] @ k[-T] * D ** -0.5
        total = np.exp(s).sum() + np.exp(own) + (N - 2000)
        assert abs(float(lse[2, 0, 0]) - np.log(total)) < 1e-4
    del big, view
    torch.cuda.empty_cache()


def test_same_bits_again_and_on_another_stream(cuda):
    from cab_attention.kernels import tree_attention
    for dt, H in (("bf16", 4), ("bf16", 32), ("fp32", 4)):
        q, k, v = (rand((2, h, n, 128), dt, n).to(cuda) for h, n in ((H, 12), (2, 5000), (2, 5000)))
        parents = torch.tensor(trees(2, 12, "tree", 3)).int().to(cuda)
        n = torch.tensor([4000, 123], dtype=torch.int32, device=cuda)
        first = tree_attention(q, k, v, parents, n, return_lse=True)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            other = tree_attention(q, k, v, parents, n, return_lse=True)
        s.synchronize()
        assert torch.equal(first[0], other[0]) and torch.equal(first[1], other[1])
