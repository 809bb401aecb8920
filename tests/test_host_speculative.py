"""Speculative decoding's entry points without a GPU: what they refuse before anything is
launched, and the cache rows a draft and a commit stand for."""

import ctypes

import numpy as np
import pytest
import torch

from cab_attention import _native as nat
from oracle import spec_oracle as S

FAKE = 0x7f0000000000  # 16-byte aligned address that is never dereferenced


def s4(*v):
    return (ctypes.c_int64 * 4)(*v)


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        from cab_attention import _build
        _build.build(verbose=False)
    return nat.load()


def test_append_at_validation(lib):
    st, big = s4(8 * 5 * 64, 5 * 64, 64, 1), s4(8 * 90 * 64, 90 * 64, 64, 1)
    call = lambda **w: lib.cab_kv_append_at(
        w.get("k", FAKE), FAKE, w.get("kd", FAKE), FAKE, w.get("es", 2), w.get("B", 1), 8, w.get("n", 5),
        w.get("D", 64), w.get("N", 90), st, st, w.get("ds", big), big, w.get("len", FAKE), None, None)
    assert call(es=1) == nat.CAB_EDTYPE
    assert call(n=-1) == nat.CAB_ESHAPE
    assert call(k=None) == nat.CAB_EINVAL
    assert call(len=None) == nat.CAB_EINVAL
    assert call(k=FAKE + 1) == nat.CAB_ESHAPE
    assert call(ds=s4(8 * 90 * 64, 90 * 64, 64, 2)) == nat.CAB_ESHAPE
    assert call(ds=s4(8 * 90 * 64, 0, 64, 1)) == nat.CAB_ESHAPE  # heads on one another
    assert b"overlap" in lib.cab_last_error()
    assert call(N=1 << 31) == nat.CAB_ESHAPE
    assert call(n=1 << 30) == nat.CAB_ESHAPE
    for empty in ("B", "n", "D", "N"):
        assert call(**{empty: 0}) == nat.CAB_OK


def test_commit_validation(lib):
    st = s4(2 * 90 * 64, 90 * 64, 64, 1)
    one = (ctypes.c_void_p * 2)(FAKE, FAKE + 4096)
    call = lambda **w: lib.cab_kv_commit(
        w.get("t", one), w.get("nt", 2), w.get("es", 2), w.get("B", 1), w.get("H", 2), w.get("N", 90), 64,
        w.get("st", st), w.get("len", FAKE), w.get("l0", 0), w.get("path", FAKE), 5, w.get("ps", 5), FAKE,
        w.get("c0", 0), w.get("new", FAKE + 64), None)
    assert call(es=3) == nat.CAB_EDTYPE
    assert call(nt=0) == nat.CAB_ESHAPE
    assert call(H=0) == nat.CAB_ESHAPE
    assert call(l0=-1) == nat.CAB_EINVAL
    assert call(l0=91) == nat.CAB_ESHAPE
    assert call(c0=-1) == nat.CAB_EINVAL
    assert call(path=None) == nat.CAB_EINVAL
    assert call(ps=4) == nat.CAB_ESHAPE
    assert call(t=(ctypes.c_void_p * 2)(FAKE, None)) == nat.CAB_EINVAL
    assert call(t=(ctypes.c_void_p * 2)(FAKE, FAKE)) == nat.CAB_EINVAL
    assert b"twice" in lib.cab_last_error()
    assert call(t=(ctypes.c_void_p * 2)(FAKE, FAKE + 1)) == nat.CAB_ESHAPE
    assert call(new=FAKE) == nat.CAB_EINVAL  # over the old lengths
    assert call(st=s4(2 * 90 * 64, 90 * 64, 32, 1)) == nat.CAB_ESHAPE
    assert call(B=70000) == nat.CAB_ESHAPE
    assert call(B=0) == nat.CAB_OK


def test_verify_validation(lib):
    st = (ctypes.c_int64 * 2)(5 * 1000, 1000)
    ws = lib.cab_verify_drafts_workspace_bytes
    need = ws(nat.CAB_BF16, 2, 5, 1000, 0, 0)
    assert need > 0 and ws(9, 2, 5, 1000, 0, 0) == 0 and ws(nat.CAB_BF16, 2, 257, 1000, 0, 0) == 0
    assert ws(nat.CAB_F32, 2, 5, 1000, 0, 1) > ws(nat.CAB_F32, 2, 5, 1000, 0, 0)
    call = lambda **w: lib.cab_verify_drafts(
        w.get("l", FAKE), w.get("d", None), w.get("dt", nat.CAB_BF16), w.get("B", 2), w.get("T", 5),
        w.get("V", 1000), st, w.get("ds", None), FAKE, w.get("p", FAKE), w.get("pl", 0), w.get("u", FAKE),
        w.get("n", FAKE), w.get("t", 1.0), FAKE, FAKE, FAKE, w.get("ws", FAKE), w.get("wsb", 1 << 30), None)
    assert call(dt=4) == nat.CAB_EDTYPE
    assert call(T=0) == nat.CAB_ESHAPE
    assert call(T=257) == nat.CAB_ESHAPE
    assert call(V=0) == nat.CAB_ESHAPE
    assert call(V=1 << 31) == nat.CAB_ESHAPE
    assert call(B=1 << 31) == nat.CAB_ESHAPE
    for t in (-1.0, float("nan"), float("inf"), 1e-7):
        assert call(t=t) == nat.CAB_EINVAL
    assert call(l=None) == nat.CAB_EINVAL
    assert call(u=None) == nat.CAB_EINVAL
    assert call(n=None) == nat.CAB_EINVAL
    assert call(d=FAKE) == nat.CAB_EINVAL  # draft strides missing
    assert call(l=FAKE + 1) == nat.CAB_ESHAPE
    assert call(pl=3) == nat.CAB_ESHAPE
    assert call(wsb=need - 1) == nat.CAB_EWORKSPACE
    assert call(ws=FAKE + 8) == nat.CAB_EWORKSPACE
    assert call(B=0) == nat.CAB_OK


def test_tree_attention_validation(lib):
    ws = lib.cab_tree_attn_workspace_bytes
    need = ws(nat.CAB_BF16, 1, 8, 2, 16, 500, 128)
    assert need > 0
    assert ws(nat.CAB_BF16, 1, 8, 3, 16, 500, 128) == 0 and ws(nat.CAB_BF16, 1, 8, 2, 257, 500, 128) == 0
    assert ws(nat.CAB_BF16, 1, 8, 2, 16, 15, 128) == 0 and ws(nat.CAB_BF16, 1, 8, 2, 16, 500, 96) == 0
    qs, ks = s4(8 * 16 * 128, 16 * 128, 128, 1), s4(2 * 500 * 128, 500 * 128, 128, 1)
    call = lambda **w: lib.cab_tree_attn_fwd(
        w.get("q", FAKE), FAKE, FAKE, w.get("dt", nat.CAB_BF16), w.get("B", 1), w.get("H", 8), w.get("Hkv", 2),
        w.get("T", 16), w.get("N", 500), w.get("D", 128), w.get("qs", qs), w.get("ks", ks), ks, qs,
        w.get("p", FAKE), w.get("pl", 0), w.get("len", None), w.get("l0", 484), w.get("scale", 0.1), FAKE, None,
        w.get("ws", FAKE), w.get("wsb", 1 << 40), None)
    assert call(dt=5) == nat.CAB_EDTYPE
    assert call(D=96) == nat.CAB_ESHAPE
    assert call(Hkv=3) == nat.CAB_ESHAPE
    assert call(T=0) == nat.CAB_ESHAPE
    assert call(T=257) == nat.CAB_ESHAPE
    assert call(N=15, l0=0) == nat.CAB_ESHAPE
    assert call(l0=485) == nat.CAB_EINVAL
    assert call(l0=-1) == nat.CAB_EINVAL
    for x in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=x) == nat.CAB_EINVAL
    assert call(p=None) == nat.CAB_EINVAL
    assert call(pl=3) == nat.CAB_ESHAPE
    assert call(q=FAKE + 2) == nat.CAB_ESHAPE
    assert call(qs=s4(8 * 16 * 128, 16 * 128, 124, 1)) == nat.CAB_ESHAPE
    assert call(ks=s4(2 * 500 * 128, 500 * 128, 128, 2)) == nat.CAB_ESHAPE
    assert call(ks=s4(1 << 40, 1 << 39, (1 << 24) + 8, 1)) == nat.CAB_ESHAPE  # past 2^25 bytes
    assert call(ks=s4(2 * 500 * 128, 500 * 128, -128, 1)) == nat.CAB_ESHAPE
    assert call(wsb=need - 1) == nat.CAB_EWORKSPACE
    assert call(ws=None) == nat.CAB_EWORKSPACE
    assert call(B=65535, Hkv=8, N=1 << 24) == nat.CAB_ESHAPE  # a list past 32 bits
    assert call(B=0) == nat.CAB_OK


def test_tree_attention_refuses_an_out_whose_rows_overlap(lib):
    qs, ks = s4(8 * 16 * 128, 16 * 128, 128, 1), s4(2 * 500 * 128, 500 * 128, 128, 1)
    call = lambda os, T=16, wsb=0: lib.cab_tree_attn_fwd(
        FAKE, FAKE, FAKE, nat.CAB_BF16, 2, 8, 2, T, 500, 128, qs, ks, ks, os, FAKE, 0, None, 484, 0.1,
        FAKE, None, FAKE, wsb, None)
    assert call(s4(0, 16 * 128, 128, 1)) == nat.CAB_ESHAPE
    assert call(s4(8 * 16 * 128, 0, 128, 1)) == nat.CAB_ESHAPE
    assert call(s4(8 * 16 * 128, 16 * 128, 64, 1)) == nat.CAB_ESHAPE
    # (the next check refuses these: a single row has no stride)
    assert call(qs) == nat.CAB_EWORKSPACE
    assert call(s4(8 * 128, 128, 0, 1), T=1) == nat.CAB_EWORKSPACE


def test_python_refusals():
    from cab_attention.cache import append_drafts, commit_drafts
    from cab_attention.kernels import tree_attention, verify_drafts
    q, k = torch.zeros(1, 4, 3, 64), torch.zeros(1, 2, 20, 64)
    up, n = torch.tensor([-1, 0, 1], dtype=torch.int32), torch.tensor([5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        tree_attention(q, k, k, up, n)
    with pytest.raises(ValueError, match="q, k and v"):
        tree_attention(q, k, k[:, :, :10], up, n)
    with pytest.raises(ValueError, match=r"\[B=1"):
        tree_attention(q, k.expand(2, 2, 20, 64), k.expand(2, 2, 20, 64), up, n)
    with pytest.raises(TypeError):
        tree_attention(q, k.half(), k.half(), up, n)
    logits, x = torch.zeros(1, 3, 10), torch.zeros(1, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU only"):
        verify_drafts(logits, x, up, temperature=0.0)
    with pytest.raises(ValueError, match=r"\[B, T, V\]"):
        verify_drafts(logits[0], x, up)
    new = torch.zeros(1, 2, 3, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        append_drafts(new, new, k, k.clone(), n)
    with pytest.raises(ValueError, match="two"):
        append_drafts(new, new[:, :, :2], k, k, n)
    with pytest.raises(ValueError, match="k_cache"):
        append_drafts(new, new, k[..., :32], k[..., :32], n)
    with pytest.raises(TypeError):
        append_drafts(new, new, k.half(), k.half(), n)
    path = torch.zeros(1, 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        commit_drafts([k], n, path, n)
    with pytest.raises(ValueError, match="at least one"):
        commit_drafts([], n, path, n)
    with pytest.raises(ValueError, match="share"):
        commit_drafts([k, k[:, :, :10]], n, path, n)
    with pytest.raises(TypeError):
        commit_drafts([k.double()], n, path, n)


def test_index32():
    t = torch.tensor([1, 2], dtype=torch.int32)
    assert nat.index32(t, "x", (2,)) is t
    assert nat.index32(torch.tensor([1, 1 << 40]), "x", (2,)).tolist() == [1, (1 << 31) - 1]
    assert nat.index32(torch.tensor([1, -(1 << 40)]), "x", (2,)).tolist() == [1, -(1 << 31)]
    assert nat.index32(torch.arange(8, dtype=torch.int32)[::2], "x", (4,)).is_contiguous()
    with pytest.raises(ValueError, match="must be"):
        nat.index32(t, "x", (3,))
    with pytest.raises(TypeError):
        nat.index32(t.float(), "x", (2,))


def test_plain_tensors_only():
    x = torch.zeros(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        nat.require_plain("op", x)
    with torch.no_grad():
        nat.require_plain("op", x)
    with pytest.raises(RuntimeError, match="plain"):
        torch.vmap(lambda t: nat.require_plain("op", t) or t)(torch.zeros(2, 3))


def test_drafted_rows_of_a_store():
    """Views and counts of drafted rows on the host (copies by torch)."""
    from cab_attention.cache.store import LayeredKV
    store = LayeredKV(initial_capacity=4)
    k = torch.arange(3.0).reshape(1, 1, 3, 1).expand(1, 2, 3, 8).contiguous()
    for layer in (0, 1):
        store.append(layer, k, k + 10)
        kk, vv = store.draft(layer, k + 100, k + 200)  # grows the buffers
        assert kk.shape[2] == 6 and store.length(layer) == 3
        assert torch.equal(kk, torch.cat([k, k + 100], 2)) and torch.equal(vv[:, :, 3:], k + 200)
        kk, _ = store.draft(layer, k[:, :, :2] + 300, k[:, :, :2])  # replaces them
        assert torch.equal(kk, torch.cat([k, k[:, :, :2] + 300], 2))
    path = torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(ValueError, match="path"):
        store.commit(torch.tensor([0, 1, 2], dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="path"):
        store.commit(path, 3)
    with pytest.raises(RuntimeError, match="GPU only"):
        store.commit(path, 1)
    assert store.length(0) == 3
    store.append(1, k, k)  # drops layer 1's drafts
    with pytest.raises(ValueError, match="same number"):
        store.commit(path, 1)
    assert torch.equal(store.view(1)[0], torch.cat([k, k], 2))


def test_oracle_lines_and_residuals():
    """The oracle itself: lines, and the draft mode's output distribution, summed exactly
    over drafts and acceptance for one draft: P(x) = q min(1, p / q) + residual = p."""
    assert S.line([-1, 0, 1, 0], 2) == [2, 1, 0] and S.line([-1, 0, -2, 2], 3) is None
    assert S.line([-1, 1], 1) is None
    p, q = np.array([0.5, 0.3, 0.2]), np.array([0.2, 0.7, 0.1])
    accept = q * np.minimum(1, p / q)
    left = np.maximum(p - q, 0)
    out = accept + (1 - accept.sum()) * left / left.sum()
    np.testing.assert_allclose(out, p, atol=1e-15)
    # ... and the path it returns takes a draft of residual weight 0 never.
    logits = np.log(np.array([[0.5, 0.5, 1e-30]] * 2))
    path, token, _ = S.verify(logits, [0, 2], [-1, 0], np.array([0, 0.5]), np.array([1.0, 2.0, 1.0]), 1.0)
    assert path == [0] and token == 0
