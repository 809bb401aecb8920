"""append_drafts and commit_drafts: rows behind each sequence's own length and the
accepted ones kept, bit for bit, whatever the strides, alignment, paths and counts;
rows that are not named keep their bits."""

import pytest
import torch

from oracle import spec_oracle as S

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def rand(shape, dt, cuda, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g).to(dt)
    x.view(-1)[::7] = float("nan")  # (copies carry any bits)
    return x.to(cuda)


def buffers(B, H, N, D, dt, cuda, seed, layout):
    if layout == "rows":      # [B, N, H, D]: heads inside a row
        return rand((B, N, H, D), dt, cuda, seed).transpose(1, 2)
    if layout == "wide":      # rows of a wider buffer
        return rand((B, H, N, D + 8), dt, cuda, seed)[..., :D]
    if layout == "odd":       # one element past a 16-byte boundary
        return rand(B * H * N * D + 1, dt, cuda, seed)[1:].view(B, H, N, D)
    return rand((B, H, N, D), dt, cuda, seed)


SHAPES = [  # B, H, n, D, N, layout
    (1, 8, 1, 128, 300, "plain"),
    (3, 2, 5, 64, 40, "plain"),
    (2, 3, 64, 128, 200, "rows"),
    (2, 1, 9, 20, 33, "plain"),   # rows of no whole 16 bytes in 16-bit types
    (4, 2, 7, 64, 50, "wide"),
    (2, 4, 33, 64, 64, "odd"),
    (1, 1, 1, 1, 1, "plain"),
    (5, 1, 130, 64, 131, "plain"),
]


@pytest.mark.parametrize("B,H,n,D,N,layout", SHAPES)
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("counted", [False, True])
def test_append(cuda, B, H, n, D, N, layout, dt, counted):
    from cab_attention.cache import append_drafts
    kc, vc = (buffers(B, H, N, D, DT[dt], cuda, s, layout) for s in (1, 2))
    k = rand((B, n, H, D), DT[dt], cuda, 3).transpose(1, 2)
    v = rand((B, H, n, D), DT[dt], cuda, 4)
    # The last lengths reach past the buffer, and one is negative.
    lengths = torch.tensor([(3 * b * N) // (2 * B) for b in range(B)], dtype=torch.int32)
    if B > 2:
        lengths[1] = -1
    counts = torch.tensor([(b + 1) * n // B for b in range(B)], dtype=torch.int32)
    want = [kc.clone(), vc.clone()]
    for new, w in ((k, want[0]), (v, want[1])):
        for b in range(B):
            at = int(lengths[b])
            if at < 0:
                continue
            m = min(int(counts[b]) if counted else n, N - at)
            if m > 0:
                w[b, :, at:at + m] = new[b, :, :m]
    versions = kc._version, vc._version
    append_drafts(k, v, kc, vc, lengths.to(cuda), counts.to(cuda) if counted else None)
    assert torch.equal(bits(kc), bits(want[0])) and torch.equal(bits(vc), bits(want[1]))
    assert kc._version > versions[0] and vc._version > versions[1]


PATHS = [  # per sequence: path, count, length
    ([0, 1, 2, -1, -1], 3, 10),   # nothing moves
    ([0, 2, 4, -1, -1], 3, 0),    # empty context
    ([0, 3, -1, -1, -1], 1, 7),   # fewer than the path holds
    ([1, 2, 3, 4, -1], 4, 5),     # each row to the one before
    ([0, 2, 2, 4, -1], 4, 3),     # not ascending: ends after two
    ([0, 5, 6, -1, -1], 3, 3),    # outside the drafts: ends after one
    ([0, 4, -1, -1, -1], 9, 11),  # count past the path
    ([0, 1, 2, 3, 4], 5, 16),     # behind the cache's end: two rows kept
    ([2, 4, -1, -1, -1], 0, 4),
    ([1, 4, -1, -1, -1], 2, -3),  # negative length
    ([4, -1, -1, -1, -1], -2, 2),
]


@pytest.mark.parametrize("layers,H,D,layout", [(1, 2, 64, "plain"), (3, 1, 128, "rows"),
                                               (35, 2, 64, "plain"), (2, 3, 20, "plain"),
                                               (2, 2, 64, "odd"), (1, 5, 64, "wide")])
@pytest.mark.parametrize("dt", list(DT))
def test_commit(cuda, layers, H, D, layout, dt):
    from cab_attention.cache import commit_drafts
    N, T, B = 18, 5, len(PATHS)
    caches = [buffers(B, H, N, D, DT[dt], cuda, s, layout) for s in range(2 * layers)]
    want, new = [c.clone() for c in caches], []
    for b, (path, count, length) in enumerate(PATHS):
        rows = S.kept(path, count, T, length, N)
        new.append(length + len(rows))
        for c, w in zip(caches, want):
            for j, f in enumerate(rows):
                w[b, :, length + j] = c[b, :, length + f]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    lengths = i32([p[2] for p in PATHS])
    got = commit_drafts(caches, lengths, i32([p[0] for p in PATHS]), i32([p[1] for p in PATHS]))
    assert got.tolist() == new and lengths.tolist() == [p[2] for p in PATHS]
    for c, w in zip(caches, want):
        assert torch.equal(bits(c), bits(w))


@pytest.mark.parametrize("T,seed", [(64, 0), (256, 1), (17, 2), (9, 3)])
def test_commit_long_paths(cuda, T, seed):
    """Paths longer than the rows a thread loads ahead, of every length."""
    from cab_attention.cache import commit_drafts
    g = torch.Generator().manual_seed(seed)
    B, H, D, N = 40, 2, 64, T + 50
    cache = torch.randn((B, H, N, D), generator=g).to(cuda)
    counts = torch.randint(0, T + 1, (B,), generator=g)
    counts[0], counts[1] = T, 8 if T > 8 else T
    path = torch.full((B, T), -1)
    for b in range(B):
        c = int(counts[b])
        path[b, :c] = torch.randperm(T, generator=g)[:c].sort().values
    lengths = torch.randint(0, 51, (B,), generator=g)
    want = cache.clone()
    for b in range(B):
        c, n = int(counts[b]), int(lengths[b])
        want[b, :, n:n + c] = cache[b][:, n + path[b, :c].to(cuda)]
    got = commit_drafts([cache], lengths.to(cuda), path.to(cuda), counts.to(cuda))  # int64
    assert torch.equal(got.cpu().long(), lengths + counts) and torch.equal(cache, want)


def test_rows_past_32_bits(cuda):
    """Offsets past 2^31 bytes and past 2^31 values within one buffer."""
    from cab_attention.cache import append_drafts, commit_drafts
    B, H, N, D = 2, 2, 5_000_000, 128
    base = torch.zeros((B, H, N, D), dtype=torch.bfloat16, device=cuda)  # 5.1 GB
    k = rand((B, H, 3, D), torch.bfloat16, cuda, 5)
    v = rand((B, H, 3, D), torch.bfloat16, cuda, 6)
    other = torch.zeros_like(base)
    lengths = torch.tensor([N - 3, N - 7], dtype=torch.int32, device=cuda)
    append_drafts(k, v, base, other, lengths)
    for b, n in enumerate((N - 3, N - 7)):
        assert torch.equal(bits(base[b, :, n:n + 3]), bits(k[b]))
        assert torch.equal(bits(other[b, :, n:n + 3]), bits(v[b]))
    path = torch.tensor([[0, 2, -1]] * 2, dtype=torch.int32, device=cuda)
    counts = torch.tensor([2, 2], dtype=torch.int32, device=cuda)
    new = commit_drafts([base, other], lengths, path, counts)
    assert new.tolist() == [N - 1, N - 5]
    for b, n in enumerate((N - 3, N - 7)):
        assert torch.equal(bits(base[b, :, n:n + 2]), bits(k[b][:, [0, 2]]))
        assert torch.equal(bits(other[b, :, n:n + 2]), bits(v[b][:, [0, 2]]))
    del base, other
    torch.cuda.empty_cache()


def test_another_stream(cuda):
    from cab_attention.cache import append_drafts, commit_drafts
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        cache = torch.zeros((1, 2, 64, 64), device=cuda)
        k = torch.randn((1, 2, 4, 64), device=cuda)
        n = torch.full((1,), 20, dtype=torch.int32, device=cuda)
        v = torch.zeros_like(cache)
        append_drafts(k, k, cache, v, n)
        path = torch.tensor([[0, 3, -1, -1]], dtype=torch.int32, device=cuda)
        n = commit_drafts([cache, v], n, path, torch.full((1,), 2, dtype=torch.int32, device=cuda))
    s.synchronize()
    assert n.tolist() == [22] and torch.equal(cache[:, :, 20:22], k[:, :, [0, 3]])
