"""Speculative decoding run together: drafts appended, attended to as a tree, verified,
and the accepted rows kept. Over ragged static buffers (eager, captured and replayed,
two streams at once) and over the evicting caches, against decoding token by token."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H, HKV, D, V, LAYERS = 4, 2, 64, 600, 3


class Model:
    """A toy of LAYERS attention layers whose q, k and v are tables over tokens (so that
    cached rows can be compared bit for bit) and whose logits are the sum of the layers'
    outputs times a matrix."""

    def __init__(self, cuda, dtype=torch.float32):
        g = torch.Generator(device=cuda).manual_seed(7)
        make = lambda *s: torch.randn(s, generator=g, device=cuda)
        self.q, self.k, self.v = (make(LAYERS, V, h, D).to(dtype) for h in (H, HKV, HKV))
        self.w = make(H * D, V) * 3 / math.sqrt(D)

    def rows(self, name, layer, tokens):  # [B, heads, T, D] as a projection leaves them
        return getattr(self, name)[layer][tokens].transpose(1, 2)

    def logits(self, outs):
        x = sum(o.float() for o in outs)
        return (x.transpose(1, 2).flatten(2) @ self.w).contiguous()


def drafts(g, cuda, pending, T, guess):
    """A tree of T nodes below each pending token: the right continuation (of ``guess``)
    hidden among wrong ones on some steps."""
    B = pending.shape[0]
    tokens = torch.randint(0, V, (B, T), generator=g, device=cuda)
    tokens[:, 0] = pending
    parents = torch.tensor([-1] + [int(i * torch.rand(1).item()) for i in range(1, T)], dtype=torch.int32)
    for b in range(B):
        node, depth = 0, 0
        for i in range(1, T):
            if int(parents[i]) == node and depth < len(guess[b]) and torch.rand(1).item() < 0.8:
                tokens[b, i] = guess[b][depth]
                node, depth = i, depth + 1
    return tokens, parents.to(cuda)


def plain_decode(model, prompt, n):
    """Greedy tokens after the prompt, one at a time in fp64 torch, and the prompt's and
    tokens' fp32 rows."""
    seq = prompt.tolist()
    for _ in range(n):
        t = torch.tensor(seq, device=prompt.device)
        x = 0
        for layer in range(LAYERS):
            q = model.q[layer][t[-1]].double()
            k, v = (getattr(model, s)[layer][t].double().repeat_interleave(H // HKV, 1) for s in "kv")
            p = torch.softmax(torch.einsum("hd,nhd->hn", q, k) / math.sqrt(D), 1)
            x = x + torch.einsum("hn,nhd->hd", p, v)
        seq.append(int((x.flatten() @ model.w.double()).argmax()))
    return seq[len(prompt):]


def ragged_step(model, keys, values, lengths, tokens, parents, uniforms, noise, temperature):
    from cab_attention.cache import append_drafts, commit_drafts
    from cab_attention.kernels import tree_attention, verify_drafts
    outs = []
    for layer in range(LAYERS):
        append_drafts(model.rows("k", layer, tokens), model.rows("v", layer, tokens), keys[layer],
                      values[layer], lengths)
        outs.append(tree_attention(model.rows("q", layer, tokens), keys[layer], values[layer], parents,
                                   lengths))
    path, counts, token = verify_drafts(model.logits(outs), tokens, parents, uniforms, noise, temperature)
    return commit_drafts(keys + values, lengths, path, counts), path, counts, token


def test_ragged_greedy_decoding(cuda):
    """Three sequences of lengths of their own, drafted right, wrong and in between: the
    tokens are those of decoding one by one, and the cached rows those tokens'."""
    torch.manual_seed(0)
    model = Model(cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    from cab_attention.cache import append_drafts
    B, N, T, want_n = 3, 160, 9, 20
    prompts = [torch.randint(0, V, (n,), generator=g, device=cuda) for n in (1, 37, 80)]
    want = [plain_decode(model, p, want_n + 12) for p in prompts]
    keys, values = ([torch.full((B, HKV, N, D), float("nan"), device=cuda) for _ in range(LAYERS)]
                    for _ in range(2))
    longest = max(len(p) for p in prompts)
    padded = torch.stack([torch.nn.functional.pad(p, (0, longest - len(p))) for p in prompts])
    # The prompt's last token is the first pending one: it is cached with the first step.
    lengths = torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device=cuda)
    for layer in range(LAYERS):
        append_drafts(model.rows("k", layer, padded), model.rows("v", layer, padded), keys[layer],
                      values[layer], torch.zeros_like(lengths), lengths)
    got = [[] for _ in range(B)]
    pending = torch.stack([p[-1] for p in prompts])
    steps = 0
    while min(len(x) for x in got) < want_n:
        tokens, parents = drafts(g, cuda, pending, T, [w[len(x):] for w, x in zip(want, got)])
        lengths, path, counts, pending = ragged_step(model, keys, values, lengths, tokens, parents, None,
                                                     None, 0.0)
        for b in range(B):
            c = int(counts[b])
            got[b] += tokens[b][path[b, 1:c].long()].tolist() + [int(pending[b])]
        steps += 1
    for b in range(B):
        assert got[b] == want[b][:len(got[b])]
        seq = torch.cat([prompts[b], torch.tensor(got[b][:-1], dtype=torch.int64, device=cuda)])
        assert int(lengths[b]) == len(seq)
        for layer in range(LAYERS):
            assert torch.equal(keys[layer][b, :, :len(seq)], model.k[layer][seq].transpose(0, 1))
            assert torch.equal(values[layer][b, :, :len(seq)], model.v[layer][seq].transpose(0, 1))
    assert steps < want_n  # (some drafts were accepted)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_captured_step(cuda, dtype, temperature):
    """A step captured once and replayed on new drafts, numbers and lengths, with eager
    steps between: every replay equals the eager step on the same inputs."""
    torch.manual_seed(1)
    model = Model(cuda, dtype)
    g = torch.Generator(device=cuda).manual_seed(2)
    B, N, T = 4, 120, 12
    fresh = lambda: [torch.randn((B, HKV, N, D), generator=g, device=cuda).to(dtype) for _ in range(LAYERS)]
    keys, values = fresh(), fresh()
    lengths = torch.tensor([0, 5, 60, 100], dtype=torch.int32, device=cuda)
    tokens, parents = drafts(g, cuda, torch.randint(0, V, (B,), generator=g, device=cuda), T, [[]] * B)
    uniforms = torch.rand((B, T), generator=g, device=cuda)
    noise = torch.empty((B, V), device=cuda).exponential_(generator=g)
    static = [lengths, tokens, parents, uniforms, noise]
    args = lambda k, v, s: (model, k, v, *s, temperature)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        ragged_step(*args([x.clone() for x in keys], [x.clone() for x in values], static))
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ragged_step(*args(keys, values, static))
    for step in range(5):
        new = [x.clone() for x in static]
        new[0] = torch.tensor([step, 100 - step, 30, 108], dtype=torch.int32, device=cuda)
        new[1], new[2] = drafts(g, cuda, torch.randint(0, V, (B,), generator=g, device=cuda), T, [[]] * B)
        new[3] = torch.rand((B, T), generator=g, device=cuda)
        new[4] = torch.empty((B, V), device=cuda).exponential_(generator=g)
        k2, v2 = [x.clone() for x in keys], [x.clone() for x in values]
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        want = ragged_step(*args(k2, v2, new))
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        for a, b in zip(keys + values, k2 + v2):
            assert torch.equal(a, b)


def test_two_streams_at_once(cuda):
    """Steps of two batches in flight on two streams give what they give alone."""
    torch.manual_seed(2)
    model = Model(cuda, torch.bfloat16)
    g = torch.Generator(device=cuda).manual_seed(3)
    B, N, T = 2, 3000, 40
    sets = []
    for i in range(2):
        keys, values = ([torch.randn((B, HKV, N, D), generator=g, device=cuda).bfloat16()
                         for _ in range(LAYERS)] for _ in range(2))
        lengths = torch.tensor([2900 - i, 17 + i], dtype=torch.int32, device=cuda)
        tokens, parents = drafts(g, cuda, torch.randint(0, V, (B,), generator=g, device=cuda), T, [[]] * B)
        noise = torch.empty((B, V), device=cuda).exponential_(generator=g)
        sets.append((keys, values, lengths, tokens, parents, torch.rand((B, T), generator=g, device=cuda),
                     noise))
    want = [ragged_step(model, [k.clone() for k in s[0]], [v.clone() for v in s[1]], *s[2:], 1.0)
            for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i] = ragged_step(model, [k.clone() for k in s[0]], [v.clone() for v in s[1]], *s[2:],
                                     1.0)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


@pytest.mark.parametrize("policy", ["cab", "h2o"])
def test_evicting_cache(cuda, policy):
    """Drafts over CABCache and H2OCache: the rows and importance totals after a commit are
    those of the accepted tokens appended one by one; evictions fall due as after as many
    updates, and keep working on what a commit left."""
    from cab_attention.cache import CABCache, H2OCache
    from cab_attention.kernels import flash_attention, key_scores, tree_attention
    torch.manual_seed(3)
    model = Model(cuda)
    g = torch.Generator(device=cuda).manual_seed(4)
    make = lambda: (CABCache if policy == "cab" else H2OCache)(max_cache_size=200, sparsity=0.5,
                                                               eviction_interval=10 ** 6)
    drafted, plain = make(), make()
    prompt = torch.randint(0, V, (1, 120), generator=g, device=cuda)
    for cache in (drafted, plain):
        for layer in range(LAYERS):
            cache.update(model.rows("k", layer, prompt), model.rows("v", layer, prompt), layer)
        cache.importance_tracker.update(torch.rand((1, 1, 1, 120), generator=torch.Generator(
            device=cuda).manual_seed(9), device=cuda))
    T = 10
    parents = torch.tensor([-1, 0, 0, 2, 1, 3, 3, 6, 2, 6], dtype=torch.int32, device=cuda)
    for step, path in enumerate(([0, 2, 3, 6], [0], [0, 1, 4], [0, 2, 3, 6, 9])):
        tokens = torch.randint(0, V, (1, T), generator=g, device=cuda)
        n = drafted.get_seq_length(0)
        query = lse = None
        for layer in range(LAYERS):
            k, v = drafted.draft(model.rows("k", layer, tokens), model.rows("v", layer, tokens), layer)
            assert k.shape[2] == n + T and drafted.get_seq_length(layer) == n
            q = model.rows("q", layer, tokens)
            out, s = tree_attention(q, k, v, parents, return_lse=True)
            if layer == 0:
                query, lse = q, s
        rows = torch.tensor([path + [-1] * (T - len(path))], dtype=torch.int32, device=cuda)
        drafted.commit(rows if step % 2 else rows[0], len(path), query, lse)
        # One by one: the same queries attend to the same keys.
        for i in path:
            t = tokens[:, i:i + 1]
            for layer in range(LAYERS):
                k, v = plain.update(model.rows("k", layer, t), model.rows("v", layer, t), layer)
                if layer == 0:
                    q = model.rows("q", 0, t)
                    _, s = flash_attention(q, k, v, return_lse=True)
                    plain.importance_tracker.add_scores(key_scores(q, k, s).sum((0, 1)))
        assert drafted.stats == plain.stats
        assert drafted.tokens_since_last_eviction == plain.tokens_since_last_eviction
        for a, b in zip(drafted.key_cache + drafted.value_cache, plain.key_cache + plain.value_cache):
            assert torch.equal(a, b)
        # (both sum split bf16 products, 2^-16 of a weight each, over 4 heads)
        torch.testing.assert_close(drafted.importance_tracker.get_scores(),
                                   plain.importance_tracker.get_scores(), atol=2e-3, rtol=0)
        assert drafted.importance_tracker.total_queries == plain.importance_tracker.total_queries
    # Past the size at which an eviction is due: one commit evicts, and drafts go on.
    before = drafted.total_evictions
    big = torch.randint(0, V, (1, 100), generator=g, device=cuda)
    for layer in range(LAYERS):
        drafted.draft(model.rows("k", layer, big), model.rows("v", layer, big), layer)
    drafted.commit(torch.arange(100, dtype=torch.int32, device=cuda), 100)
    assert drafted.total_evictions == before + 1 and drafted.get_seq_length(0) == drafted.keep_size
    tokens = torch.randint(0, V, (1, 3), generator=g, device=cuda)
    kept = [k.clone() for k in drafted.key_cache]
    for layer in range(LAYERS):
        drafted.draft(model.rows("k", layer, tokens), model.rows("v", layer, tokens), layer)
    drafted.commit(torch.tensor([[1, 2, -1]], dtype=torch.int32, device=cuda), 2)
    for layer in range(LAYERS):
        want = torch.cat([kept[layer], model.rows("k", layer, tokens)[:, :, 1:3]], 2)
        assert torch.equal(drafted.key_cache[layer], want)
    for layer in range(LAYERS):
        drafted.draft(model.rows("k", layer, tokens), model.rows("v", layer, tokens), layer)
    drafted.commit(torch.tensor([-1, -1, -1], dtype=torch.int32, device=cuda), 0)
    assert drafted.get_seq_length(0) == drafted.keep_size + 2


def test_evicting_cache_of_a_batch(cuda):
    """Two sequences with paths of their own and one count; odd widths and bf16."""
    from cab_attention.cache import LayeredKV
    g = torch.Generator(device=cuda).manual_seed(6)
    store = LayeredKV(initial_capacity=3)
    make = lambda n: torch.randn((2, 3, n, 20), generator=g, device=cuda).bfloat16()
    want = []
    for layer in range(2):
        k, v, dk, dv = make(5), make(5), make(6), make(6)
        store.append(layer, k, v)
        store.draft(layer, dk, dv)
        want.append([torch.cat([x, torch.stack([d[0][:, [0, 2, 5]], d[1][:, [0, 1, 3]]])], 2)
                     for x, d in ((k, dk), (v, dv))])
    store.commit(torch.tensor([[0, 2, 5, -1, -1, -1], [0, 1, 3, 4, -1, -1]], device=cuda), 3)  # int64
    for layer in range(2):
        k, v = store.view(layer)
        assert torch.equal(k, want[layer][0]) and torch.equal(v, want[layer][1])


def test_refusals_on_the_device(cuda):
    from cab_attention.cache import LayeredKV, append_drafts, commit_drafts
    from cab_attention.kernels import tree_attention, verify_drafts
    cache = torch.zeros((1, 2, 20, 64), device=cuda)
    n = torch.zeros(1, dtype=torch.int32, device=cuda)
    path = torch.zeros((1, 3), dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="twice"):
        commit_drafts([cache, cache], n, path, n)
    with pytest.raises(ValueError, match="overlap"):
        commit_drafts([cache[:, :1].expand(1, 2, 20, 64)], n, path, n)
    with pytest.raises(RuntimeError, match="no gradient"):
        commit_drafts([cache.clone().requires_grad_()], n, path, n)
    with torch.inference_mode():
        closed = torch.zeros((1, 2, 20, 64), device=cuda)
    with pytest.raises(RuntimeError, match="inference"):
        commit_drafts([closed], n, path, n)
    with pytest.raises(RuntimeError, match="GPU only"):
        commit_drafts([cache], n.cpu(), path, n)
    new = torch.zeros((1, 2, 3, 64), device=cuda)
    with pytest.raises(RuntimeError, match="inference"):
        append_drafts(new, new, closed, closed.clone(), n)
    with pytest.raises(RuntimeError, match="no gradient"):
        append_drafts(new.clone().requires_grad_(), new, cache, cache.clone(), n)
    q = torch.zeros((1, 4, 3, 64), device=cuda)
    up = torch.tensor([-1, 0, 1], device=cuda)
    with pytest.raises(RuntimeError, match="no gradient"):
        tree_attention(q.clone().requires_grad_(), cache, cache, up, n)
    with pytest.raises(ValueError, match="out must match"):
        tree_attention(q, cache, cache, up, n, out=q.half())
    with pytest.raises(ValueError, match="scale"):
        tree_attention(q, cache, cache, up, n, scale=-1.0)
    with pytest.raises(ValueError, match="lengths"):
        tree_attention(q, cache, cache, up, torch.zeros(2, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError, match="at least as many rows"):
        tree_attention(q, cache[:, :, :2], cache[:, :, :2], up)
    logits = torch.zeros((1, 3, 9), device=cuda)
    tokens = torch.zeros((1, 3), dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError, match="uniforms and noise"):
        verify_drafts(logits, tokens, up)
    with pytest.raises(ValueError, match="noise"):
        verify_drafts(logits, tokens, up, logits[:, :, 0], logits[:, 0, :3])
    with pytest.raises(ValueError, match="temperature"):
        verify_drafts(logits, tokens, up, logits[:, :, 0], logits[:, 0], temperature=-1.0)
    with pytest.raises(TypeError):
        verify_drafts(logits, tokens.float(), up, temperature=0)
    with pytest.raises(ValueError, match="draft_logits"):
        verify_drafts(logits, tokens, up, logits[:, :, 0], logits[:, 0], draft_logits=logits.half())
    store = LayeredKV()
    store.append(0, new.requires_grad_(), new.detach())
    store.draft(0, new.detach(), new.detach())
    with pytest.raises(RuntimeError, match="no gradient"):
        store.commit(path[0], 1)

