"""Decoding over a paged cache without a GPU: what the entry points refuse before anything is
launched, the frequencies of rotary positions, and the oracle against closed forms."""

import ctypes
import math

import numpy as np
import pytest
import torch

from cab_attention import CABAttention, _native as nat
from cab_attention.cache import append_paged
from cab_attention.kernels import Rotary, adjust_logits, paged_attention
from oracle import paged_oracle as P

FAKE = 0x7f0000000000  # 16-byte aligned address that is never dereferenced


def arr(*v):
    return (ctypes.c_int64 * len(v))(*v)


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        from cab_attention import _build
        _build.build(verbose=False)
    return nat.load()


def test_rotary_validation(lib):
    far = FAKE + (1 << 36)
    ptrs = lambda *p: (ctypes.c_void_p * len(p))(*p)
    st = (8 * 100 * 64, 100 * 64, 64, 1)
    kv = (2 * 100 * 64, 100 * 64, 64, 1)
    call = lambda **w: lib.cab_rotary(
        w.get("n", 2), w.get("x", ptrs(FAKE, FAKE + (1 << 30))), w.get("out", ptrs(far, far + (1 << 30))),
        w.get("dt", nat.CAB_BF16), w.get("B", 2), w.get("heads", arr(8, 2)), w.get("N", 100),
        w.get("D", 64), w.get("xs", arr(*st, *kv)), w.get("os", arr(*st, *kv)), None, w.get("pl", 0),
        w.get("turns", FAKE), w.get("R", 64), 0, w.get("a", 1.0), 0, None)
    assert call(dt=7) == nat.CAB_EDTYPE
    for n in (0, 3):
        assert call(n=n) == nat.CAB_ESHAPE
    for R in (0, 63, 66, -2):
        assert call(R=R) == nat.CAB_ESHAPE
    assert call(D=514, R=2) == nat.CAB_ESHAPE
    assert call(turns=None) == nat.CAB_EINVAL
    for a in (float("nan"), float("inf")):
        assert call(a=a) == nat.CAB_EINVAL
    assert call(heads=arr(-1, 2)) == nat.CAB_ESHAPE
    assert call(x=ptrs(None, FAKE)) == nat.CAB_EINVAL
    assert call(x=ptrs(FAKE + 1, FAKE + (1 << 30))) == nat.CAB_ESHAPE
    assert call(xs=arr(*st[:3], 2, *kv)) == nat.CAB_ESHAPE
    assert call(os=arr(8 * 100 * 64, 100 * 64, 32, 1, *kv)) == nat.CAB_ESHAPE
    assert b"overlap" in lib.cab_last_error()
    assert call(out=ptrs(far, far)) == nat.CAB_EINVAL           # q's and k's results meet
    assert call(out=ptrs(FAKE + 128, far)) == nat.CAB_EINVAL    # into q, shifted
    assert call(out=ptrs(FAKE + (1 << 30), far)) == nat.CAB_EINVAL  # q's result into k
    assert call(B=1 << 20, N=16) == nat.CAB_ESHAPE              # 2^24 tokens
    for empty in ("B", "N"):
        assert call(**{empty: 0}) == nat.CAB_OK
    assert call(heads=arr(0, 0)) == nat.CAB_OK


def test_append_validation(lib):
    new, pool = arr(2 * 5 * 64, 5 * 64, 64, 1), arr(2 * 16 * 64, 16 * 64, 64, 1)
    qs = arr(8 * 5 * 64, 5 * 64, 64, 1)
    call = lambda **w: lib.cab_paged_append(
        w.get("k", FAKE), FAKE + (1 << 20), w.get("kp", FAKE + (1 << 32)), w.get("vp", FAKE + (1 << 33)),
        w.get("q", FAKE + (1 << 21)), w.get("qo", FAKE + (1 << 22)), w.get("dt", nat.CAB_BF16), w.get("B", 3),
        w.get("H", 8), w.get("Hkv", 2), w.get("n", 5), w.get("D", 64), w.get("pages", 40), w.get("S", 16), new,
        w.get("vs", new), w.get("ps", pool), pool, w.get("qs", qs), qs, w.get("table", FAKE), w.get("tl", 12),
        w.get("M", 12), w.get("len", FAKE), None, None, w.get("pl", 0), w.get("turns", FAKE), w.get("R", 64), 0,
        w.get("a", 1.0), None)
    assert call(dt=5) == nat.CAB_EDTYPE
    for bad in (dict(n=-1), dict(Hkv=0), dict(H=-1), dict(S=0), dict(D=0), dict(D=513), dict(R=3), dict(R=66),
                dict(tl=11), dict(M=1 << 28), dict(n=1 << 23), dict(k=FAKE + 1),
                dict(vs=arr(2 * 5 * 64, 5 * 64, 64, 2)), dict(ps=arr(2 * 16 * 64, 16 * 64, 32, 1))):
        assert call(**bad) == nat.CAB_ESHAPE, bad
    for bad in (dict(k=None), dict(kp=None), dict(table=None), dict(len=None), dict(turns=None), dict(q=None),
                dict(qs=None), dict(a=math.nan), dict(vp=FAKE + (1 << 32) + 64), dict(kp=FAKE + 64),
                dict(qo=FAKE + (1 << 21) + 2), dict(qo=FAKE + (1 << 32))):
        assert call(**bad) == nat.CAB_EINVAL, bad
    for empty in ("B", "n"):
        assert call(**{empty: 0}) == nat.CAB_OK


def test_attention_validation(lib):
    ws = lib.cab_paged_attn_workspace_bytes
    need = ws(nat.CAB_BF16, 3, 8, 2, 500, 16, 128)
    assert need > 0 and ws(9, 3, 8, 2, 500, 16, 128) == 0
    assert ws(0, 3, 8, 3, 500, 16, 128) == 0 and ws(0, 3, 8, 2, 500, 16, 96) == 0
    assert ws(0, 3, 8, 2, 1 << 30, 16, 64) == 0
    qs, pool = arr(8 * 128, 128, 128, 1), arr(2 * 16 * 128, 16 * 128, 128, 1)
    call = lambda **w: lib.cab_paged_attn_fwd(
        w.get("q", FAKE), w.get("k", FAKE + (1 << 32)), FAKE + (1 << 33), w.get("dt", nat.CAB_BF16),
        w.get("B", 3), w.get("H", 8), w.get("Hkv", 2), w.get("D", 128), w.get("pages", 900), w.get("S", 16),
        w.get("qs", qs), w.get("ks", pool), pool, w.get("os", qs), w.get("table", FAKE), w.get("tl", 500),
        w.get("M", 500), w.get("len", FAKE), w.get("scale", 0.1), w.get("out", FAKE + (1 << 20)), None,
        w.get("ws", FAKE), w.get("wsb", 1 << 40), None)
    assert call(dt=5) == nat.CAB_EDTYPE
    for bad in (dict(D=96), dict(Hkv=3), dict(Hkv=0), dict(S=0), dict(M=-1), dict(pages=-1), dict(tl=499),
                dict(B=70000), dict(M=1 << 28), dict(pages=1 << 31), dict(q=FAKE + 2),
                dict(qs=arr(8 * 128, 124, 128, 1)), dict(qs=arr(8 * 128, 128, 128, 2)),
                dict(ks=arr(2 * 16 * 128, 16 * 128, -128, 1)), dict(ks=arr(1 << 40, 1 << 39, (1 << 24) + 8, 1)),
                dict(os=arr(8 * 128, 64, 128, 1))):
        assert call(**bad) == nat.CAB_ESHAPE, bad
    for bad in (dict(q=None), dict(k=None), dict(table=None), dict(len=None), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(out=FAKE + 256),
                dict(out=FAKE + (1 << 32))):
        assert call(**bad) == nat.CAB_EINVAL, bad
    assert call(wsb=need - 1) == nat.CAB_EWORKSPACE
    assert call(ws=None) == nat.CAB_EWORKSPACE
    assert call(B=0) == nat.CAB_OK


def test_adjust_validation(lib):
    st = arr(5 * 1000, 1000)
    call = lambda **w: lib.cab_adjust_logits(
        w.get("l", FAKE), w.get("out", FAKE + (1 << 24)), w.get("dt", nat.CAB_BF16), w.get("B", 2), w.get("T", 5),
        w.get("V", 1000), st, w.get("os", st), w.get("h", FAKE), w.get("L", 70), w.get("hl", 70), None, None,
        None, w.get("r", 1.1), None, w.get("p", 0.0), None, w.get("f", 0.0), w.get("bt", FAKE), FAKE,
        w.get("n", 3), w.get("bl", 3), w.get("al", None), w.get("as", None), w.get("d", None), w.get("par", None),
        w.get("pl", 0), None)
    assert call(dt=4) == nat.CAB_EDTYPE
    for bad in (dict(T=-1), dict(V=-1), dict(L=-1), dict(n=-1), dict(V=1 << 31), dict(L=1 << 31),
                dict(T=257, d=FAKE, par=FAKE), dict(d=FAKE, par=FAKE, pl=3), dict(l=FAKE + 1),
                dict(os=arr(5 * 1000, 500)), dict(B=1 << 24)):
        assert call(**bad) == nat.CAB_ESHAPE, bad
    for bad in (dict(l=None), dict(h=None), dict(hl=69), dict(bt=None), dict(bl=2), dict(al=FAKE),
                dict(d=FAKE), dict(r=0.0), dict(r=-1.0), dict(r=math.nan), dict(r=math.inf), dict(p=math.nan),
                dict(f=math.inf), dict(out=FAKE + 16)):
        assert call(**bad) == nat.CAB_EINVAL, bad
    for empty in ("B", "T", "V"):
        assert call(**{empty: 0}) == nat.CAB_OK


SCALINGS = [None, dict(type="linear", factor=4.0), dict(type="ntk", factor=2.5),
            dict(type="yarn", factor=4.0, original_length=4096),
            dict(type="yarn", factor=16.0, original_length=8192, beta_fast=24.0, beta_slow=2.0, amplitude=1.25),
            dict(type="bands", factor=8.0, original_length=8192),
            dict(type="bands", factor=3.0, original_length=2048, low=2.0, high=9.0)]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["type"] if s else "none")
@pytest.mark.parametrize("dim, base", [(2, 10000.0), (32, 500000.0), (64, 10000.0), (128, 10000.0)])
def test_frequencies_and_turns(scaling, dim, base):
    if dim == 2 and scaling and scaling["type"] == "ntk":
        pytest.skip("one pair has no base")
    r = Rotary(128, rotary_dim=dim, base=base, scaling=scaling)
    f, amplitude = P.rotary_frequencies(dim, base, scaling)
    np.testing.assert_allclose(r.frequencies, f, rtol=1e-14)
    assert r.amplitude == pytest.approx(amplitude, rel=1e-14)
    # 2^64 of them are a turn: p * turns modulo 2^64 is the angle, for any p.
    for t, x in zip(r.turns.tolist(), r.frequencies):
        for p in (1, 77777, 10 ** 9, -12345):
            angle = (p * t % 2 ** 64) / 2.0 ** 64 * 2 * math.pi
            # A frequency is rounded to 2^-65 of a turn, which p multiplies (1e9: 1.7e-10 rad);
            # the comparison's own product |p x| is off by half a step of 53 bits, twice.
            off = abs(p) * 2 * math.pi * 2.0 ** -65 + abs(p * x) * 2.0 ** -52
            assert abs(np.exp(1j * angle) - np.exp(1j * (p * x))) < 1e-14 + off
    assert not r.state_dict() and r.half().turns.dtype is torch.int64


@pytest.mark.parametrize("bad", [
    dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=33), dict(head_dim=64, rotary_dim=0),
    dict(head_dim=513), dict(head_dim=514), dict(head_dim=64, base=1.0), dict(head_dim=64, base=math.nan),
    dict(head_dim=64, scaling=dict(type="other", factor=2.0)), dict(head_dim=64, scaling=dict(factor=2.0)),
    dict(head_dim=64, scaling=dict(type="linear")), dict(head_dim=64, scaling=dict(type="linear", factor=0.0)),
    dict(head_dim=64, scaling=dict(type="linear", factor=2.0, low=1.0)),
    dict(head_dim=64, scaling=dict(type="yarn", factor=2.0)),
    dict(head_dim=64, scaling=dict(type="yarn", factor=2.0, original_length=100, amplitude=math.inf)),
    dict(head_dim=64, scaling=dict(type="bands", factor=2.0, original_length=100, low=4.0, high=4.0))])
def test_rotary_refuses_at_construction(bad):
    with pytest.raises(ValueError):
        Rotary(**bad)


def test_attention_module_refuses_another_head_dim():
    with pytest.raises(ValueError, match="rotary"):
        CABAttention(512, 8, rotary=Rotary(128))
    with pytest.raises(ValueError, match="positions"):
        CABAttention(512, 8)(torch.zeros(1, 64, 512), positions=torch.arange(64))


def test_tensors_on_the_host_are_refused():
    q, pages = torch.zeros(2, 8, 1, 64), torch.zeros(5, 2, 16, 64)
    table, lengths = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(2, 2, 1, 64)
    for call in (lambda: Rotary(64)(q), lambda: paged_attention(q, pages, pages, table, lengths),
                 lambda: append_paged(kv, kv, pages, pages.clone(), table, lengths),
                 lambda: adjust_logits(torch.zeros(2, 1, 100))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_shapes_and_types_are_refused_on_the_host():
    q, pages = torch.zeros(2, 8, 1, 64), torch.zeros(5, 2, 16, 64)
    table, lengths = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(2, 2, 1, 64)
    rot = Rotary(64)
    for error, call in (
            (ValueError, lambda: rot(q[..., :32])), (ValueError, lambda: rot(q, kv[:1])),
            (TypeError, lambda: rot(q, kv.half())), (ValueError, lambda: rot(q[0])),
            (ValueError, lambda: paged_attention(q[:, :, 0], pages, pages, table, lengths)),
            (ValueError, lambda: paged_attention(q.expand(-1, -1, 2, -1), pages, pages, table, lengths)),
            (ValueError, lambda: paged_attention(q[..., :32], pages, pages, table, lengths)),
            (ValueError, lambda: paged_attention(q, pages, pages[:4], table, lengths)),
            (TypeError, lambda: paged_attention(q, pages.half(), pages, table, lengths)),
            (ValueError, lambda: append_paged(kv, kv[:1], pages, pages, table, lengths)),
            (ValueError, lambda: append_paged(kv, kv, pages[:, :1], pages[:, :1], table, lengths)),
            (TypeError, lambda: append_paged(kv.half(), kv, pages, pages, table, lengths)),
            (ValueError, lambda: adjust_logits(torch.zeros(2, 100)))):
        with pytest.raises(error):
            call()


# ---------------------------------------------------------------------------
# The oracle
# ---------------------------------------------------------------------------

def test_oracle_rotary_turns_pairs():
    x = np.zeros((1, 1, 1, 4))
    x[0, 0, 0, 0] = 2.0
    for inter, second in ((True, 1), (False, 2)):
        y = P.rotary(x, np.array([[3]]), np.array([math.pi / 6, 1.0]), 1.5, inter)  # a quarter turn
        want = np.zeros(4)
        want[second] = 3.0
        np.testing.assert_allclose(y[0, 0, 0], want, atol=1e-15)
        np.testing.assert_allclose(P.rotary(y, np.array([[3]]), np.array([math.pi / 6, 1.0]), 1 / 1.5, inter,
                                            inverse=True), x, atol=1e-15)


def test_oracle_pages_are_a_cache_in_pieces():
    rng = np.random.default_rng(0)
    pages, new = rng.normal(size=(7, 2, 4, 8)), rng.normal(size=(1, 2, 5, 8))
    table = np.array([[5, 2, 6]])
    got = P.append(pages, new, table, np.array([3]))
    whole = got[[5, 2, 6]].transpose(1, 0, 2, 3).reshape(2, 12, 8)
    np.testing.assert_array_equal(whole[:, 3:8], new[0])
    np.testing.assert_array_equal(whole[:, :3], pages[5][:, :3])
    np.testing.assert_array_equal(np.delete(got, [5, 2], 0), np.delete(pages, [5, 2], 0))
    q = rng.normal(size=(1, 2, 1, 8))
    out, lse = P.attention(q, got, got, table, np.array([8]))
    z = torch.tensor(q[0]) @ torch.tensor(whole[:, :8]).transpose(1, 2) / math.sqrt(8)
    np.testing.assert_allclose(out[0], torch.softmax(z, -1) @ torch.tensor(whole[:, :8]), rtol=1e-12)
    np.testing.assert_allclose(lse[0], torch.logsumexp(z, -1), rtol=1e-12)


def test_oracle_adjust_by_hand():
    x = np.array([[[2.0, -2.0, 1.0, 0.5, 3.0]]])
    y = P.adjust(x, np.array([[0, 1, 1, 2, 2, 9]]), np.array([5]), np.array([2]), 2.0, 0.25, 0.5,
                 np.array([[3, 3]]), np.array([[7.0, 1.0]]), np.array([[[True, True, True, True, False]]]))
    # 0: prompt; 1: prompt and once; 2: twice; 3: bias (the last one); 4: not allowed
    np.testing.assert_array_equal(y[0, 0], [1.0, -4.75, -0.75, 1.5, -np.inf])
    y = P.adjust(np.zeros((1, 3, 4)), drafts=np.array([[0, 1, 2]]), parents=np.array([[-1, 0, 0]]), presence=1.0)
    np.testing.assert_array_equal(y[0], [[-1, 0, 0, 0], [-1, -1, 0, 0], [-1, 0, -1, 0]])
