"""paged_attention against the float64 oracle: at the edges of its cuts (32-key steps, 128-key
pieces, 16-key blocks), of pages and of row tiles (16, 32 rows a K / V head), with pages that are
not there, and with values that must not reach a row."""

import math

import numpy as np
import pytest
import torch

from cab_attention.kernels import paged_attention
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# Each weight's rounding to 16 bits moves an output, a mean of values of up to about 5, by at
# most half a step (bf16 2^-9 of the weight), and so does the output's own rounding (of a value up to
# about 4): together below 2 * 5 * 2^-9 (bf16), 2 * 5 * 2^-12 (fp16); fp32: sums of D + some 256
# terms, each off by 2^-24. The log-sum-exp is fp32 throughout: scores of up to about 8, their sums and the
# exponentials' errors, 2^-24 each.
ATOL = {"bf16": 2e-2, "fp16": 2.5e-3, "fp32": 2e-5}
LSE_ATOL = 2e-5


def rand(shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(DT[dt])


def np64(t):
    return t.detach().double().cpu().numpy()


def setup(B, H, Hkv, D, S, lengths, dt, cuda, seed=0, columns=None, gone=0.0):
    """Pages in any order; what is behind a length or in free pages is NaN."""
    rng = np.random.default_rng(seed)
    columns = columns or max(1, -(-max(max(lengths), 1) // S))
    pages = B * columns + 3
    table = rng.permutation(pages)[:B * columns].reshape(B, columns)
    k, v = (torch.full((pages, Hkv, S, D), float("nan"), dtype=DT[dt]) for _ in range(2))
    for b in range(B):
        n = min(max(lengths[b], 0), columns * S)
        for pool, x in ((k, rand((Hkv, n, D), dt, 10 * b + 1)), (v, rand((Hkv, n, D), dt, 10 * b + 2))):
            for i in range(-(-n // S)):
                m = min(S, n - i * S)
                pool[table[b, i], :, :m] = x[:, i * S:i * S + m]
    table[rng.random(table.shape) < gone] = -1
    q = rand((B, 1, H, D), dt, 5, 1.5).transpose(1, 2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    return (q, k, v, table), (q.to(cuda), k.to(cuda), v.to(cuda), i32(table), i32(lengths))


def check(host, got, lengths, dt, scale=None):
    q, k, v, table = host
    out, lse = P.attention(np64(q), np64(k), np64(v), table, lengths, scale)
    gone = np.isneginf(lse)
    assert np.array_equal(np.isneginf(np64(got[1])), gone)
    np.testing.assert_allclose(np64(got[1])[~gone], lse[~gone], atol=LSE_ATOL, rtol=0)
    np.testing.assert_allclose(np64(got[0]), out, atol=ATOL[dt], rtol=0)
    assert not np64(got[0])[gone].any()


CASES = [  # B, H, H_kv, S, lengths
    (1, 4, 4, 16, [1]),                       # one key
    (3, 8, 2, 16, [0, 15, 16]),               # nothing; around a block
    (4, 4, 1, 16, [17, 31, 32, 33]),          # around a step
    (3, 4, 2, 64, [127, 128, 129]),           # around a piece
    (2, 2, 2, 16, [511, 512]),                # the longest that a workgroup takes whole
    (2, 8, 2, 16, [513, 700]),                # split
    (3, 16, 1, 32, [1500, 3, 0]),             # a full row tile; a split unit beside short ones
    (1, 17, 1, 16, [900]),                    # 17 rows: the second row tile's kernel
    (1, 33, 1, 48, [2000]),                   # 33 rows: two row tiles
    (2, 6, 3, 1, [40, 700]),                  # a key a page
    (2, 6, 3, 5, [33, 1201]),                 # pages that end inside a block
    (3, 4, 4, 24, [24, 600, 23]),             # and inside a step
    (2, 34, 1, 20, [650, 7]),                 # 34 rows, pages off the blocks
    (1, 2, 1, 256, [5000]),                   # large pages; more than 32 steps a wave
    (1, 1, 1, 16, [20000]),                   # many partials
    (70, 2, 1, 16, [(37 * i) % 200 for i in range(70)]),   # more than 64 sequences
    (80, 4, 4, 16, [600 + (91 * i) % 50 for i in range(80)]),  # units over workgroups' borders
    (2, 4, 2, 16, [-7, 5]),                   # a negative length
    (3, 2, 1, 16, [639, 640, 641]),           # around what a workgroup takes whole of a few units
    (3, 2, 1, 16, [0, 640, 600]),
    (2, 2, 1, 16, [200, 130]),                # the same in fp32, D = 128
    (2, 2, 1, 8, [208, 7]),
    (2, 2, 1, 16, [400, 130]),                # and D = 64
    (2, 2, 1, 8, [408, 390]),
    (64, 8, 4, 16, [1024 - 16 * (i % 3) for i in range(64)]),  # the same of a unit a CU
    (70, 4, 2, 16, [(97 * i) % 1100 for i in range(70)]),      # a list of more than 64 sequences
    (130, 4, 4, 16, [(31 * i) % 1200 for i in range(130)]),    # and of two workgroups a CU
    (40, 40, 1, 16, [(211 * i) % 900 for i in range(40)]),     # three row tiles over one list
]


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", CASES, ids=lambda c: str(c[:4]))
def test_against_the_oracle(cuda, case, dt, D):
    B, H, Hkv, S, lengths = case
    host, args = setup(B, H, Hkv, D, S, lengths, dt, cuda)
    check(host, paged_attention(*args, return_lse=True), lengths, dt)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("S", [16, 64, 7])
@pytest.mark.parametrize("lengths", [[100, 300, 64], [3000, 50, 2999]], ids=str)
def test_pages_that_are_gone(cuda, S, dt, lengths):
    host, args = setup(3, 8, 2, 128, S, lengths, dt, cuda, gone=0.4)
    check(host, paged_attention(*args, return_lse=True), lengths, dt)
    q, k, v, table, n = args
    bad = table.clone().long()
    bad[bad < 0] = torch.tensor([k.shape[0], -5, 2 ** 40], device=cuda)[torch.arange(int((bad < 0).sum()), device=cuda) % 3]
    a, b = paged_attention(q, k, v, bad, n.long(), return_lse=True), paged_attention(*args, return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("S", [1, 2, 4, 8, 24, 12, 6, 5])
def test_pages_of_other_sizes(cuda, S, dt):
    """Sizes whose blocks of one page are of 8, 4, 2 and 1 keys: whole and in parts, pages gone."""
    for lengths in ([70, 33, 1], [1500, 7, 1111]):
        host, args = setup(3, 4, 2, 128, S, lengths, dt, cuda, gone=0.2)
        check(host, paged_attention(*args, return_lse=True), lengths, dt)


@pytest.mark.parametrize("S, n", [(16, 18500), (32, 18500), (8, 9500), (4, 5000), (3, 4000)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_stretches_past_a_look_up(cuda, S, n, dt):
    """64 sequences over a few pages in any order, so that a wave takes more steps than its lanes hold the
    pages of (32 of them with whole blocks of 16 keys, 16 of 8, 8 of 4, 2 of odd sizes)."""
    rng = np.random.default_rng(S)
    pool, lengths = 61, [n - 37 * b for b in range(64)]
    table = rng.integers(-3, pool, (64, -(-n // S)))
    q, k, v = rand((64, 2, 1, 128), dt, 1, 1.5), rand((pool, 1, S, 128), dt, 2), rand((pool, 1, S, 128), dt, 3)
    got = paged_attention(*(x.to(cuda) for x in (q, k, v)), torch.tensor(table, device=cuda),
                          torch.tensor(lengths, device=cuda), return_lse=True)
    check((q, k, v, table), got, lengths, dt)


def test_queries_of_any_strides(cuda):
    """Values apart from one another, rows off 16-byte boundaries, heads and sequences broadcast."""
    _, (q, k, v, table, n) = setup(2, 8, 2, 64, 16, [90, 33], "bf16", cuda)
    apart = q.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    off = torch.zeros(2, 8, 1, 67, dtype=q.dtype, device=cuda)[..., 3:].copy_(q)
    for x in (apart, off, q[:1].expand_as(q), q[:, :1].expand_as(q)):
        out, lse = paged_attention(x, k, v, table, n, return_lse=True)
        a, b = paged_attention(x.contiguous(), k, v, table, n, return_lse=True)
        assert torch.equal(out, a) and torch.equal(lse, b)


def test_nothing_to_see(cuda):
    """All pages gone, no columns, no pages, lengths of zero: 0 and -inf, for short and long tables."""
    for columns in (3, 200):
        _, (q, k, v, table, n) = setup(2, 8, 2, 64, 16, [40, 48], "bf16", cuda, columns=columns)
        for t, m in ((torch.full_like(table, -1), n), (table, n * 0), (table, n * 0 - 3), (table[:, :0], n)):
            out, lse = paged_attention(q, k, v, t, m, return_lse=True)
            assert not out.any() and torch.isneginf(lse).all()
        out, lse = paged_attention(q, k[:0], v[:0], table, n, return_lse=True)
        assert not out.any() and torch.isneginf(lse).all()
    assert paged_attention(q[:0], k, v, table[:0], n[:0]).shape == (0, 8, 1, 64)


def test_lengths_past_the_table(cuda):
    host, (q, k, v, table, n) = setup(2, 4, 2, 64, 16, [160, 70], "fp16", cuda)
    check(host, paged_attention(q, k, v, table, torch.tensor([2 ** 31 - 1, 70], device=cuda), return_lse=True),
          [160, 70], "fp16")


@pytest.mark.parametrize("columns", [None, 100])
@pytest.mark.parametrize("dt", list(DT))
def test_scores_without_a_softmax(cuda, dt, columns):
    """NaN or +inf among the scores, or all -inf: NaN for both results, in that row alone; single -inf
    scores weigh nothing."""
    host, args = setup(2, 4, 2, 64, 16, [70, 90], dt, cuda, columns=columns)
    q, k, v, table, n = args
    clean = paged_attention(*args, return_lse=True)
    page = int(table[0, 1])
    for value, at in ((float("nan"), 3), (float("inf"), 4)):
        k2 = k.clone()
        k2[page, 0, at, 7] = value
        out, lse = paged_attention(q, k2, v, table, n, return_lse=True)
        sign = np.sign(np64(q)[0, :2, 0, 7])
        for h in range(2):
            if value != value or sign[h] > 0:  # +inf score
                assert torch.isnan(out[0, h]).all() and torch.isnan(lse[0, h]).all()
            else:                              # -inf score: a key less
                assert torch.isfinite(out[0, h]).all() and float(lse[0, h]) < float(clean[1][0, h])
        assert torch.equal(out[0, 2:], clean[0][0, 2:]) and torch.equal(out[1], clean[0][1])
    k2, q2 = k.clone(), q.clone()
    q2[..., 0] = 1.0
    for i in range(5):
        k2[int(table[0, i]), 0, :, 0] = -float("inf")
    out, lse = paged_attention(q2, k2, v, table, n, return_lse=True)
    assert torch.isnan(out[0, :2]).all() and torch.isnan(lse[0, :2]).all()
    assert torch.isfinite(out[0, 2:]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("dt", list(DT))
def test_wide_scores(cuda, dt):
    """One key far above all others, at each edge in turn: its V row, its score."""
    host, (q, k, v, table, n) = setup(1, 4, 1, 128, 16, [1300], dt, cuda)
    for key in (0, 15, 16, 31, 127, 128, 1279, 1299):
        k2 = k.clone()
        k2[int(table[0, key // 16]), 0, key % 16] = q[0, 0, 0] * 40
        out, lse = paged_attention(q, k2, v, table, n, return_lse=True)
        row = v[int(table[0, key // 16]), 0, key % 16]
        # The key's weight is 2^(s c - level) with the level s c rounded to 24 bits (of up to 2000: 1.2e-4), not
        # 1. In fp32 product and sum hold the same weight: their roundings and the quotient's, 4
        # half steps. In 16 bits the weight is rounded in the product and not in the sum: half
        # a step and 1.2e-4 ln 2 more, and the output's own half step.
        eps = torch.finfo(DT[dt]).eps
        rtol = 4 * 2.0 ** -24 if dt == "fp32" else eps + 1e-4
        np.testing.assert_allclose(np64(out)[0, 0, 0], np64(row), rtol=rtol, atol=0)
        want = (np64(q)[0, 0, 0] * np64(k2)[int(table[0, key // 16]), 0, key % 16]).sum() * 128 ** -0.5
        assert abs(float(lse[0, 0]) - want) < 64 * 2.0 ** -24 * abs(want) + 1e-6


def test_layouts_scale_and_out(cuda):
    """Pools laid out [P, S, H, D] with K and V side by side, a table that is a part of a larger one,
    another scale, q itself as out, the same bits again."""
    host, (q, k, v, table, n) = setup(3, 8, 2, 64, 16, [700, 3, 90], "bf16", cuda)
    want = paged_attention(q, k, v, table, n, scale=0.3, return_lse=True)
    check(host, want, [700, 3, 90], "bf16", 0.3)
    both = torch.stack((k.transpose(1, 2), v.transpose(1, 2)), 3)  # [P, S, H, 2, D]
    kp, vp = both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2)
    big = torch.full((5, table.shape[1] + 2), 7, dtype=torch.int32, device=cuda)
    big[1:4, 2:] = table
    rows = q.transpose(1, 2).contiguous()  # [B, 1, H, D]
    got = paged_attention(rows.transpose(1, 2), kp, vp, big[1:4, 2:], n, 0.3, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    room = torch.zeros((3, 8, 2, 64), dtype=torch.bfloat16, device=cuda)
    out = room[:, :, 1:]
    assert paged_attention(q, k, v, table, n, 0.3, out=out) is out and torch.equal(out, want[0])
    assert not room[:, :, 0].any() and out._version > 0
    own = q.contiguous().clone()
    paged_attention(own, k, v, table, n, 0.3, out=own)
    assert torch.equal(own, want[0])
    odd = torch.zeros((3, 8, 1, 65), dtype=torch.bfloat16, device=cuda)[..., 1:]
    odd.copy_(q)
    assert torch.equal(paged_attention(odd, k, v, table, n, 0.3), want[0])


def test_shared_pages(cuda):
    """Sequences with one prefix, and one page twice in a sequence."""
    host, (q, k, v, table, n) = setup(2, 4, 2, 64, 16, [64, 64], "fp32", cuda)
    shared = host[3].copy()
    shared[1, :3] = shared[0, :3]
    shared[0, 3] = shared[0, 0]
    got = paged_attention(q, k, v, torch.tensor(shared, dtype=torch.int32, device=cuda), n, return_lse=True)
    check((*host[:3], shared), got, [64, 64], "fp32")


def test_same_bits_whatever_memory_held(cuda):
    host, args = setup(3, 8, 2, 128, 16, [900, 3, 2100], "bf16", cuda)
    first = paged_attention(*args, return_lse=True)
    for value in (float("nan"), float("inf"), 3.0):
        junk = torch.full((8 << 20,), value, device=cuda)
        del junk  # the workspace is taken from here
        again = paged_attention(*args, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 bytes, and pages at its far end."""
    S, D, Hkv = 64, 128, 2
    pages = (1 << 32) // (Hkv * S * D * 2) + 70
    pool = torch.empty((pages, Hkv, S, D), dtype=torch.bfloat16, device=cuda)
    pool.fill_(float("nan"))
    table = torch.tensor([[pages - 1, 0, pages - 30], [1, pages - 2, 2]], dtype=torch.int32)
    k = rand((2, 3, Hkv, S, D), "bf16", 1)
    pool[table.to(cuda).long()] = k.to(cuda)
    q = rand((2, 4, 1, D), "bf16", 2, 1.5)
    lengths = torch.tensor([192, 150], dtype=torch.int32)
    got = paged_attention(q.to(cuda), pool, pool, table.to(cuda), lengths.to(cuda), return_lse=True)
    small = torch.arange(6, dtype=torch.int32).view(2, 3)
    want = paged_attention(q.to(cuda), k.view(6, Hkv, S, D).to(cuda), k.view(6, Hkv, S, D).to(cuda),
                           small.to(cuda), lengths.to(cuda), return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals_on_the_device(cuda):
    _, (q, k, v, table, n) = setup(2, 4, 2, 64, 16, [64, 30], "bf16", cuda)
    for args, kw, error, match in (
            ((q[..., :32], k[..., :32], v[..., :32], table, n), {}, ValueError, "D must be"),
            ((q[:, :3], k, v, table, n), {}, ValueError, "multiple"),
            ((q, k, v, table[:1], n), {}, ValueError, "page_table"),
            ((q, k, v, table, n[:1]), {}, ValueError, "lengths"),
            ((q, k, v, table.float(), n), {}, TypeError, "page_table"),
            ((q, k, v, table, n), dict(scale=0.0), ValueError, "scale"),
            ((q, k, v, table, n), dict(out=q[:, :2]), ValueError, "out"),
            ((q, k, v, table, n), dict(out=k[:2, :1, :4].transpose(1, 2)), ValueError, "shares memory"),
            ((q, k.transpose(2, 3).contiguous().transpose(2, 3), v, table, n), {}, ValueError, "stride"),
            ((q.clone().requires_grad_(), k, v, table, n), {}, RuntimeError, "gradient"),
            ((q.double(), k.double(), v.double(), table, n), {}, TypeError, "dtype")):
        with pytest.raises(error, match=match):
            paged_attention(*args, **kw)


@pytest.mark.parametrize("dt", list(DT))
def test_scores_without_a_softmax_over_parts(cuda, dt):
    """The same where several workgroups share the sequence: NaN or infinite keys in any part, a NaN
    query, NaN in a V row, all scores -inf, and pages gone but for one part."""
    host, (q, k, v, table, n) = setup(2, 4, 2, 64, 16, [3000, 2500], dt, cuda)
    clean = paged_attention(q, k, v, table, n, return_lse=True)
    check(host, clean, [3000, 2500], dt)
    q = q.clone()
    q[..., 0] = 1.0
    clean = paged_attention(q, k, v, table, n, return_lse=True)
    for key in (0, 1500, 2999):
        page, place = int(table[0, key // 16]), key % 16
        for value in (float("nan"), float("inf")):
            k2 = k.clone()
            k2[page, 0, place, 0] = value
            out, lse = paged_attention(q, k2, v, table, n, return_lse=True)
            assert torch.isnan(out[0, :2]).all() and torch.isnan(lse[0, :2]).all()
            assert torch.equal(out[0, 2:], clean[0][0, 2:]) and torch.equal(out[1], clean[0][1])
            assert torch.equal(lse[0, 2:], clean[1][0, 2:]) and torch.equal(lse[1], clean[1][1])
        v2 = v.clone()
        v2[page, 0, place, 9] = float("nan")
        out, lse = paged_attention(q, k, v2, table, n, return_lse=True)
        assert torch.isnan(out[0, :2, 0, 9]).all() and torch.equal(lse, clean[1])
        assert int(torch.isnan(out).sum()) == 2
    k2 = k.clone()
    k2[table[0].long(), 0, :, 0] = -float("inf")
    out, lse = paged_attention(q, k2, v, table, n, return_lse=True)
    assert torch.isnan(out[0, :2]).all() and torch.isnan(lse[0, :2]).all() and torch.equal(out[0, 2:], clean[0][0, 2:])
    q2 = q.clone()
    q2[1, 3, 0, 5] = float("nan")
    out, lse = paged_attention(q2, k, v, table, n, return_lse=True)
    assert torch.isnan(out[1, 3]).all() and torch.isnan(lse[1, 3]).all()
    assert torch.equal(out[0], clean[0][0]) and torch.equal(out[1, :3], clean[0][1, :3])
    for kept in (0, 90, 187):  # one page left of sequence 0
        t = table.clone()
        t[0] = -1
        t[0, kept] = table[0, kept]
        got = paged_attention(q, k, v, t, n, return_lse=True)
        check((q.cpu(), host[1], host[2], t.cpu().numpy()), got, [3000, 2500], dt)


@pytest.mark.parametrize("dt", list(DT))
def test_values_that_are_infinite(cuda, dt):
    """An infinity in a V row that is seen is the output's, whole and over parts."""
    for n in (40, 3000):
        host, (q, k, v, table, m) = setup(1, 2, 1, 64, 16, [n], dt, cuda)
        q.zero_()  # all weights alike, and a power of two relative to the level: nothing left of them
        v2 = v.clone()
        v2[int(table[0, 1]), 0, 3, 7] = -float("inf")
        out = paged_attention(q, k, v2, table, m)
        assert torch.isneginf(out[0, :, 0, 7]).all() and int((~torch.isfinite(out)).sum()) == 2


def test_values_near_the_types_end(cuda):
    """The least weights times the largest values: 300 keys of weight 1 and of V = 0, and one whose weight is a
    power of two (nothing is left of its upper bits) and whose V is 2^127."""
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device=cuda)
    k, v = (torch.zeros(20, 1, 16, 64, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    q[..., 0], k[3, 0, 5, 0], v[3, 0, 5] = 1.0, -112.0, 2.0 ** 127
    table = torch.arange(20, dtype=torch.int32, device=cuda)[None]
    n = torch.tensor([301], dtype=torch.int32, device=cuda)
    out = paged_attention(q, k, v, table, n, scale=math.log(2.0))
    # (an output's half step; the weight's exponent, 112 in fp32, and its power, 2^-17; the rest's 2^-126 of 2^-112)
    want = 2.0 ** (127 - 112) / 300
    assert (out.double() / want - 1).abs().max() <= 2.0 ** -8 + 2.0 ** -14


# An output's own rounding, and what is left of the weights': 16-bit weights in two parts keep 16 bits
# (bf16: 8 and 8, a step of 2^-16 of the weight) or 22 (fp16).
@pytest.mark.parametrize("dt, rest", [("bf16", 2.0 ** -15), ("fp16", 2.0 ** -20), ("fp32", 0.0)])
@pytest.mark.parametrize("case", [(2, 8, 2, 16, [600, 31]), (2, 8, 2, 16, [5000, 700]), (2, 8, 1, 24, [900, 7])], ids=str)
def test_only_the_output_is_rounded(cuda, case, dt, rest):
    B, H, Hkv, S, lengths = case
    host, args = setup(B, H, Hkv, 128, S, lengths, dt, cuda)
    out, _ = P.attention(*(np64(x) for x in host[:3]), host[3], lengths)
    mean, _ = P.attention(np64(host[0]), np64(host[1]), np.abs(np64(host[2])), host[3], lengths)
    # (and of fp32 sums of D + some 256 terms, 2^-24 each of the mean of |v|)
    off = np.abs(np64(paged_attention(*args)) - out)
    assert (off <= np.abs(out) * torch.finfo(DT[dt]).eps / 2 * (1 + 1e-6) + mean * (rest + 400 * 2.0 ** -24)
            + torch.finfo(DT[dt]).tiny).all()
