"""What EvictingCache.commit and LayeredKV.commit refuse leaves the cache as it was: rows,
lengths, drafts, importance totals and statistics."""

import copy

import pytest
import torch

import cab_attention.cache.store as store_module
from cab_attention.cache import CABCache, LayeredKV

T, N, H, HKV, D = 5, 12, 4, 2, 64


def filled(device, batches=(2, 2), dtype=torch.float32):
    """A cache of one layer per entry of ``batches``, N rows and T drafts each."""
    g = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(s, generator=g).to(device, dtype)
    cache = CABCache(max_cache_size=1000, sparsity=0.5, eviction_interval=10 ** 6)
    for layer, b in enumerate(batches):
        cache.update(make(b, HKV, N, D), make(b, HKV, N, D), layer)
        cache.draft(make(b, HKV, T, D), make(b, HKV, T, D), layer)
    if device != "cpu":
        cache.importance_tracker.update(torch.rand((1, 1, 1, N), generator=g).to(device))
    q = make(batches[0], H, T, D)
    return cache, q, torch.zeros((batches[0], H, T), device=device)


def state(cache):
    out = [copy.deepcopy(cache.stats), cache.tokens_since_last_eviction, cache.total_evictions,
           cache.importance_tracker.total_queries]
    tensors = []
    for L in cache._store.layers:
        out += [L.length, L.drafted]
        tensors += [x[:, :, :L.length + L.drafted].clone() for x in (L.k, L.v)]
    if cache.importance_tracker.get_scores() is not None:
        tensors.append(cache.importance_tracker.get_scores().clone())
    return out, tensors


def same(a, b):
    return a[0] == b[0] and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))


PATH = torch.tensor([[0, 2, 3, -1, -1], [0, 1, 4, -1, -1]], dtype=torch.int32)

# What a caller may get wrong, of (path, query, lse, scale).
WRONG = {
    "query dtype": lambda p, q, s: (p, q.half(), s, None),
    "query double": lambda p, q, s: (p, q.double(), s, None),
    "heads": lambda p, q, s: (p, q[:, :3], s[:, :3], None),
    "batch of query": lambda p, q, s: (p, q[:1], s[:1], None),
    "head dim": lambda p, q, s: (p, torch.cat([q, q], 3), s, None),
    "lse dtype": lambda p, q, s: (p, q, s.half(), None),
    "lse shape": lambda p, q, s: (p, q, s[:, :, :2], None),
    "no lse": lambda p, q, s: (p, q, None, None),
    "scale": lambda p, q, s: (p, q, s, -1.0),
    "scale nan": lambda p, q, s: (p, q, s, float("nan")),
    "path batch": lambda p, q, s: (p[:1], q, s, None),
    "path nodes": lambda p, q, s: (p[:, :4], q[:, :, :4], s[:, :, :4], None),
    "path dims": lambda p, q, s: (p[None], q, s, None),
    "path type": lambda p, q, s: (p.float(), q, s, None),
}


@pytest.mark.parametrize("name", list(WRONG))
def test_no_row_moves_on_the_host(monkeypatch, name):
    """The copy that would move rows is not reached."""
    cache, q, lse = filled("cpu")
    moved = []
    monkeypatch.setattr(store_module, "commit_rows", lambda *a: moved.append(a))
    before = state(cache)
    path, q, lse, scale = WRONG[name](PATH, q, lse)
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        cache.commit(path, 3, q, lse, scale)
    assert not moved and same(state(cache), before)


def test_groups_are_checked_first_on_the_host(monkeypatch):
    store = LayeredKV()
    for layer, b in enumerate((2, 3)):
        x = torch.randn(b, HKV, N, D)
        store.append(layer, x, x)
        store.draft(layer, x[:, :, :T], x[:, :, :T])
    moved = []
    monkeypatch.setattr(store_module, "commit_rows", lambda *a: moved.append(a))
    for path, count in ((PATH, 3), (PATH, 0), (PATH, -1), (PATH, 6)):
        with pytest.raises(ValueError, match="path must"):
            store.commit(path, count)
    assert not moved and [(L.length, L.drafted) for L in store.layers] == [(N, T)] * 2


def test_key_scores_refuses_keys_of_another_batch_or_head_dim():
    """(Its kernel would read past them.)"""
    from cab_attention.kernels import key_scores
    q, k, lse = torch.zeros(2, H, T, D), torch.zeros(2, HKV, N, D), torch.zeros(2, H, T)
    for bad in (k[:1], k[..., :32], k[0]):
        with pytest.raises(ValueError, match="k must be"):
            key_scores(q, bad, lse)
    with pytest.raises(RuntimeError, match="GPU only"):
        key_scores(q, k, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(WRONG) + ["lse device", "query device", "second batch", "gradients"])
def test_refused_commits_change_nothing(cuda, name):
    cache, q, lse = filled(cuda, (2, 3) if name == "second batch" else (2, 2))
    path, scale = PATH.to(cuda), None
    if name == "lse device":
        bad = path, q, lse.cpu(), None
    elif name == "query device":
        bad = path, q.cpu(), lse.cpu(), None
    elif name in ("second batch", "gradients"):
        bad = path, q, lse, None
    else:
        bad = WRONG[name](path, q, lse)
    if name == "gradients":  # (the second layer's buffers would record them)
        cache._store.layers[1].v.requires_grad_()
    before = state(cache)
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        cache.commit(bad[0], 3, *bad[1:])
    assert same(state(cache), before)
    # The right call afterwards is taken.
    if name == "gradients":
        cache._store.layers[1].v.requires_grad_(False)
    if name == "second batch":
        path = path[0]
    cache.commit(path, 3, q, lse, scale)
    assert cache.get_seq_length(0) == cache.get_seq_length(1) == N + 3
    assert cache.importance_tracker.total_queries == before[0][3] + 3
    for layer, L in enumerate(cache._store.layers):
        k = before[1][2 * layer]
        rows = path if path.dim() == 2 else path.expand(k.shape[0], T)
        for b in range(k.shape[0]):
            keep = list(range(N)) + [N + x for x in rows[b, :3].tolist()]
            assert torch.equal(L.k[b, :, :N + 3], k[b][:, keep])
