"""Calls whose writes would share memory are refused: rows of one tensor whose strides, each wide
enough by itself, meet, and tensors that lie in one another. What is only interleaved is taken."""

import ctypes

import pytest

from cab_attention import _native as nat

FAKE = 0x7f0000000000  # 16-byte aligned address that is never dereferenced


def s4(*v):
    return (ctypes.c_int64 * 4)(*v)


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        from cab_attention import _build
        _build.build(verbose=False)
    return nat.load()


D = 64
# Strides of [2, 3, 4] rows of 64 values; which of them are apart.
STRIDES = {
    (3 * 4 * D, 4 * D, D): True,          # contiguous
    (3 * 4 * D, D, 3 * D): True,          # heads inside a row
    (D, 2 * D, 6 * D): True,              # sequences inside
    (5000, 1600, 400): True,              # gaps
    (D, D, D): False,
    (3 * 4 * D, D, D): False,             # heads and rows alike
    (4 * D, 4 * D, D): False,             # sequences and heads alike
    (8 * D, 4 * D, D): False,             # a sequence's last head on the next one's
    (3 * 4 * D, 3 * D, D): False,         # a head's last row on the next one's
    (3 * 4 * D, 4 * D, D - 8): False,
    (1 << 62, 4 * D, D): False,           # nothing is that far
}


@pytest.mark.parametrize("st", list(STRIDES))
def test_rows_of_one_tensor(lib, st):
    apart, st = STRIDES[st], s4(*st, 1)
    plain = s4(3 * 4 * D, 4 * D, D, 1)
    # (apart: the next thing that is wrong is found; nothing is launched)
    got = lib.cab_tree_attn_fwd(FAKE, FAKE, FAKE, nat.CAB_BF16, 2, 3, 3, 4, 4, D, plain, plain, plain, st,
                                FAKE, 0, None, 0, 0.1, FAKE, None, FAKE, 0, None)
    assert got == (nat.CAB_EWORKSPACE if apart else nat.CAB_ESHAPE)
    assert apart or b"overlap" in lib.cab_last_error()
    if not apart:
        one = (ctypes.c_void_p * 1)(FAKE)
        assert lib.cab_kv_commit(one, 1, 2, 2, 3, 4, D, st, FAKE, 0, FAKE, 5, 5, FAKE, 0, FAKE + 64,
                                 None) == nat.CAB_ESHAPE
        assert b"overlap" in lib.cab_last_error()
        for k, v in ((st, plain), (plain, st)):
            assert lib.cab_kv_append_at(FAKE, FAKE, FAKE, FAKE + (1 << 20), 2, 2, 3, 4, D, 4, plain, plain,
                                        k, v, FAKE, None, None) == nat.CAB_ESHAPE
            assert b"overlap" in lib.cab_last_error()


# Pairs of [2, 3, 4] rows of 64 values (strides, offset of the second in values): which of them
# share memory. Alike layouts are told apart place by place, others by their spans.
FUSED = (3 * 4 * 2 * D, 4 * 2 * D, 2 * D)
WIDE = (3 * 4 * 5 * D, 4 * 5 * D, 5 * D)
PLAIN = (3 * 4 * D, 4 * D, D)
HEADS_INSIDE = (3 * 4 * D, D, 3 * D)
UNEVEN = (60 * D, 18 * D, 5 * D)                 # the next head is three rows' places and 3 D on
PAIRS = [
    (UNEVEN, UNEVEN, 3 * D, True),
    (UNEVEN, UNEVEN, 2 * D, False),
    (UNEVEN, UNEVEN, -4 * D, False),
    (PLAIN, PLAIN, 0, True),
    (PLAIN, PLAIN, D, True),                     # one row on
    (PLAIN, PLAIN, -4 * D, True),
    (PLAIN, PLAIN, 2 * 3 * 4 * D, False),        # one behind the other
    (PLAIN, PLAIN, -2 * 3 * 4 * D, False),
    (PLAIN, PLAIN, 2 * 3 * 4 * D - 8, True),
    (FUSED, FUSED, D, False),                    # K and V side by side in each row
    (FUSED, FUSED, -D, False),
    (FUSED, FUSED, D - 8, True),
    (FUSED, FUSED, 2 * D, True),                 # the next row's
    (FUSED, FUSED, 3 * D, False),
    (WIDE, WIDE, 4 * D, False),
    (WIDE, WIDE, 4 * D + 8, True),               # reaches into the next row
    (WIDE, WIDE, 3 * 4 * 5 * D - 4 * D, False),
    (HEADS_INSIDE, HEADS_INSIDE, 2 * D, True),
    (PLAIN, HEADS_INSIDE, 0, True),
    (PLAIN, HEADS_INSIDE, 2 * 3 * 4 * D, False),
    (FUSED, PLAIN, D, True),                     # (their spans meet)
]


SHARED = [p[:3] for p in PAIRS if p[3]]
APART = [p[:3] for p in PAIRS if not p[3]]


@pytest.mark.parametrize("ks,vs,offset", SHARED)
@pytest.mark.parametrize("es", [2, 4])
def test_append_refuses_buffers_that_share(lib, ks, vs, offset, es):
    plain = s4(*PLAIN, 1)
    assert lib.cab_kv_append_at(FAKE, FAKE + 4096, FAKE, FAKE + es * offset, es, 2, 3, 4, D, 4, plain, plain,
                                s4(*ks, 1), s4(*vs, 1), FAKE, None, None) == nat.CAB_EINVAL
    assert b"share memory" in lib.cab_last_error()


def in_one_memory(cuda, dt, ks, vs, offset):
    """Two caches of such a layout in one tensor."""
    import torch
    g = torch.Generator().manual_seed(1)
    memory = torch.randn(20000, generator=g).to(dt).to(cuda)
    base = 8000 - offset // 2 // 8 * 8
    view = lambda m, st, at: m.as_strided((2, 3, 4, D), (*st, 1), at)
    return memory, lambda m: (view(m, ks, base), view(m, vs, base + offset))


@pytest.mark.gpu
@pytest.mark.parametrize("ks,vs,offset", APART)
@pytest.mark.parametrize("dt", ["bfloat16", "float32"])
def test_append_takes_buffers_that_are_apart(cuda, dt, ks, vs, offset):
    import torch
    from cab_attention.cache import append_drafts
    dt = getattr(torch, dt)
    memory, caches = in_one_memory(cuda, dt, ks, vs, offset)
    k, v = torch.randn((2, 2, 3, 2, D), device=cuda).to(dt)
    want = memory.clone()
    for cache, new in zip(caches(want), (k, v)):
        cache[0, :, 1:3], cache[1, :, 2:4] = new[0], new[1]
    append_drafts(k, v, *caches(memory), torch.tensor([1, 2], dtype=torch.int32, device=cuda))
    assert torch.equal(memory, want)


@pytest.mark.gpu
def test_append_of_one_tensor_as_both(cuda):
    import torch
    from cab_attention.cache import append_drafts
    cache, k = torch.zeros((1, 2, 9, D), device=cuda), torch.randn((1, 2, 3, D), device=cuda)
    n = torch.tensor([4], dtype=torch.int32, device=cuda)
    append_drafts(k, k, cache, cache, n)
    assert torch.equal(cache[:, :, 4:7], k) and not cache[:, :, 7:].any()
    with pytest.raises(ValueError, match="share memory"):
        append_drafts(k, k + 1, cache, cache, n)


def commit_status(lib, st, addresses, es=2):
    ptrs = (ctypes.c_void_p * len(addresses))(*addresses)
    return lib.cab_kv_commit(ptrs, len(addresses), es, 2, 3, 4, D, s4(*st, 1), FAKE, 0, FAKE, 5, 5, FAKE, 0,
                             FAKE + 64, None)


@pytest.mark.parametrize("st,offset", [(a, o) for a, b, o in SHARED if a == b and o])
@pytest.mark.parametrize("es", [2, 4])
def test_commit_refuses_tensors_that_share(lib, st, offset, es):
    far = [FAKE + es * 100000 * (i + 1) for i in range(5)]
    for at in ([FAKE, FAKE + es * offset], far + [far[2] + es * offset], [far[3] - es * offset] + far):
        assert commit_status(lib, st, at, es) == nat.CAB_EINVAL
        assert b"share memory" in lib.cab_last_error()
    assert commit_status(lib, st, far + [far[0]], es) == nat.CAB_EINVAL
    assert b"twice" in lib.cab_last_error()
    # Side by side in each row, but for one that is not.
    if st == WIDE:
        row = [FAKE + es * D * i for i in (3, 0, 4, 1)]
        assert commit_status(lib, st, row + [FAKE + es * (2 * D + 8)], es) == nat.CAB_EINVAL
        assert b"share memory" in lib.cab_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("st,offset", [(a, o) for a, b, o in APART if a == b])
@pytest.mark.parametrize("dt", ["bfloat16", "float32"])
def test_commit_takes_tensors_that_are_apart(cuda, dt, st, offset):
    import torch
    from cab_attention.cache import commit_drafts
    memory, caches = in_one_memory(cuda, getattr(torch, dt), st, st, offset)
    want = memory.clone()
    for c in caches(want):
        c[0, :, 1:3], c[1, :, 0] = c[0][:, [2, 3]].clone(), c[1][:, 1].clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    path = i32([[1, 2, -1], [1, -1, -1]])
    assert commit_drafts(caches(memory), i32([1, 0]), path, i32([2, 1])).tolist() == [3, 1]
    assert torch.equal(memory, want)


@pytest.mark.gpu
def test_commit_of_layers_side_by_side(cuda):
    """70 layers' rows in one tensor [B, H, N, layer, D]: two launches."""
    import torch
    from cab_attention.cache import commit_drafts
    memory = torch.randn((2, 1, 9, 70, D), device=cuda)
    want = memory.clone()
    want[0, :, 5], want[1, :, 2] = memory[0, :, 7], memory[1, :, 3]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    new = commit_drafts(memory.unbind(3), i32([4, 2]), i32([[0, 3, -1, -1], [1, -1, -1, -1]]), i32([2, 1]))
    assert new.tolist() == [6, 3] and torch.equal(memory, want)


def tree_status(lib, q, k, v, out, q_st, kv_st, out_st, T=4):
    """tree_attention of [2, 3, T, D] queries over [2, 3, 40, D] caches, everything else right (a call
    that is not refused would be launched: only for refusals)."""
    return lib.cab_tree_attn_fwd(q, k, v, nat.CAB_F32, 2, 3, 3, T, 40, D, s4(*q_st, 1), s4(*kv_st, 1),
                                 s4(*kv_st, 1), s4(*out_st, 1), FAKE, 0, None, 0, 0.1, out, None, FAKE,
                                 1 << 40, None)


def test_tree_attention_refuses_an_out_among_its_inputs(lib):
    cache, size = (3 * 40 * D, 40 * D, D), 2 * 3 * 40 * D * 4
    q, k, v, far = FAKE, FAKE + (1 << 24), FAKE + (1 << 25), FAKE + (1 << 26)
    heads = (4 * 3 * D, D, 3 * D)
    expanded = (0, 40 * D, D)
    for out, q_st, kv_st, out_st in (
            (q, PLAIN, cache, heads),              # q's memory in another order
            (q + 4 * D, PLAIN, cache, PLAIN),      # a row on
            (k, PLAIN, cache, PLAIN), (v, PLAIN, cache, PLAIN),
            (k + size - 256, PLAIN, cache, PLAIN), # its last row
            (k + size // 2 - 256, PLAIN, expanded, PLAIN),
            (far - 4 * D, (0, 0, 0), cache, PLAIN)):
        at = far if q_st == (0, 0, 0) else q
        assert tree_status(lib, at, k, v, out, q_st, kv_st, out_st) == nat.CAB_EINVAL
        assert b"out shares memory" in lib.cab_last_error()


@pytest.mark.gpu
def test_tree_attention_writes_over_q(cuda):
    """out may be q itself, and lie beside q and between the caches' rows."""
    import torch
    from cab_attention.kernels import tree_attention
    for dt, H, T in ((torch.float32, 2, 5), (torch.bfloat16, 4, 30), (torch.float16, 4, 64)):
        fused = torch.randn((2, T, 3 * H, D), device=cuda).to(dt)
        q, beside = fused[:, :, :H].transpose(1, 2), fused[:, :, H:2 * H].transpose(1, 2)
        k, v = (torch.randn((2, 2, 400, D), device=cuda).to(dt) for _ in range(2))
        up = torch.tensor([-1] + [i // 2 for i in range(T - 1)], dtype=torch.int32, device=cuda)
        want = tree_attention(q, k, v, up)
        rest = fused[:, :, 2 * H:].clone()
        assert torch.equal(tree_attention(q, k, v, up, out=beside), want) and torch.equal(beside, want)
        assert torch.equal(tree_attention(q, k, v, up, out=q), want) and torch.equal(q, want)
        assert torch.equal(fused[:, :, 2 * H:], rest)
        with pytest.raises(ValueError, match="shares memory"):
            tree_attention(q, k, v, up, out=fused[:, :, 1:H + 1].transpose(1, 2))
        if H == 2:
            with pytest.raises(ValueError, match="shares memory"):
                tree_attention(q, k, v, up, out=k[:, :, 100:100 + T])


def test_tree_attention_of_the_most_rows(lib):
    """B H T = 2^26 rows need one thread more than a launch takes, and the three numbers below it
    as many."""
    ws = lib.cab_tree_attn_workspace_bytes
    st = s4(64, 64, 64, 1)
    for B, H, T in ((1 << 13, 1 << 7, 1 << 6), (1 << 10, 1 << 8, 1 << 8), (8191, 8193, 1), (18631, 3602, 1)):
        assert B * H * T in (1 << 26, (1 << 26) - 1, (1 << 26) - 2)
        assert ws(nat.CAB_BF16, B, H, H, T, T, D) == 0
        assert lib.cab_tree_attn_fwd(FAKE, FAKE, FAKE, nat.CAB_BF16, B, H, H, T, T, D, st, st, st, st, FAKE, 0,
                                     None, 0, 0.1, FAKE, None, FAKE, 1 << 40, None) == nat.CAB_ESHAPE
        assert b"too large" in lib.cab_last_error()
    assert 16380 * 4097 == (1 << 26) - 4 and ws(nat.CAB_BF16, 16380, 4097, 4097, 1, 1, D) > 0
