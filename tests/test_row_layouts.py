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
