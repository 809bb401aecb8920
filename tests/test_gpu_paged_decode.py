"""Decoding over a paged cache as a program does it: prompts appended, then steps of rotated and
appended keys, attention over the pages, adjusted logits and a sampled token; against a float64
loop, with pages evicted on the way, and captured into a graph."""

import numpy as np
import pytest
import torch

from cab_attention.cache import append_paged
from cab_attention.kernels import Rotary, adjust_logits, flash_attention, paged_attention, verify_drafts
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

L, B, H, HKV, D, V, S, PAGES, COLUMNS = 2, 3, 4, 2, 64, 501, 16, 30, 8
PROMPTS = [37, 1, 48]
STEPS = 8


class Model:
    """Two layers of attention alone, tied embeddings; weights in fp32, or as float64 arrays."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s, k=1.0: k * torch.randn(s, generator=g)
        dim = H * D
        self.embed = r(V, dim)
        self.wq = [r(dim, H * D, k=dim ** -0.5) for _ in range(L)]
        self.wk = [r(dim, HKV * D, k=dim ** -0.5) for _ in range(L)]
        self.wv = [r(dim, HKV * D, k=dim ** -0.5) for _ in range(L)]
        self.wo = [r(H * D, dim, k=dim ** -0.5) for _ in range(L)]
        self.prompts = [torch.randint(0, V, (n,), generator=g) for n in PROMPTS]
        self.noise = [torch.empty(B, V).exponential_(generator=g) for _ in range(STEPS + 1)]

    def to(self, f):
        out = Model.__new__(Model)
        out.__dict__ = {k: [f(x) for x in v] if isinstance(v, list) else f(v) for k, v in self.__dict__.items()}
        return out


def evicted(table, step):
    """After some steps sequence 2 loses its second page, sequence 0 its first."""
    if step == 3:
        table[2, 1] = -1
    if step == 5:
        table[0, 0] = -1


def oracle_loop(m, rot, repetition, presence, temperature, table):
    """Every sequence by itself, every step from all of its rows anew."""
    f, amplitude = P.rotary_frequencies(rot.rotary_dim, rot.base, rot.scaling)
    pages = np.zeros((L, 2, PAGES, HKV, S, D))
    turn = lambda x, n: P.rotary(x, n + np.arange(x.shape[2])[None], f, amplitude, rot.interleaved)
    heads = lambda x, n: x.reshape(1, -1, n, D).transpose(0, 2, 1, 3)
    table = table.copy()
    tokens, logits = [], []
    histories = [list(p) for p in m.prompts]
    for step in range(-1, STEPS):
        evicted(table, step)
        row, chosen = [], []
        for b in range(B):
            new = histories[b] if step < 0 else histories[b][-1:]
            n0 = len(histories[b]) - len(new)
            outs = []
            for i, token in enumerate(new):  # token by token: a prompt, too
                x = m.embed[int(token)][None]
                for layer in range(L):
                    q, k, v = (heads(x @ w[layer], n) for w, n in ((m.wq, H), (m.wk, HKV), (m.wv, HKV)))
                    at = [n0 + i]
                    for kind, rows in ((0, turn(k, at[0])), (1, v)):
                        pages[layer, kind] = P.append(pages[layer, kind], rows, table[b:b + 1], at)
                    o, _ = P.attention(turn(q, at[0]), pages[layer, 0], pages[layer, 1], table[b:b + 1], [at[0] + 1])
                    x = x + o.transpose(0, 2, 1, 3).reshape(1, H * D) @ m.wo[layer]
                outs.append(x)
            z = (outs[-1] @ m.embed.T) * 0.1
            z = P.adjust(z[None], np.array([histories[b]]), prompts=[PROMPTS[b]], repetition=repetition, presence=presence)
            w = np.exp(z[0, 0] / temperature - (z[0, 0] / temperature).max())
            row.append(z[0, 0])
            chosen.append(int(np.argmax(w / m.noise[step + 1][b])))
        for b in range(B):
            histories[b].append(chosen[b])
        tokens.append(chosen)
        logits.append(row)
    return np.array(tokens), np.array(logits)


def kernel_loop(m, rot, repetition, presence, temperature, table, cuda):
    pools = [[torch.zeros((PAGES, HKV, S, D), device=cuda) for _ in range(2)] for _ in range(L)]
    table = torch.tensor(table, dtype=torch.int32, device=cuda)
    history = torch.zeros((B, COLUMNS * S), dtype=torch.int32, device=cuda)
    prompt = torch.tensor(PROMPTS, dtype=torch.int32, device=cuda)
    most = max(PROMPTS)
    first = torch.zeros((B, most), dtype=torch.int64, device=cuda)
    for b, p in enumerate(m.prompts):
        history[b, :len(p)] = p.int()
        first[b, :len(p)] = p
    heads = lambda x, n: x.view(B, -1, n, D).transpose(1, 2)
    root, ones = torch.tensor([-1], dtype=torch.int32, device=cuda), torch.zeros((B, 1), device=cuda)
    # Prompts: padded, causal attention over the rows at hand, and appended with counts.
    x, none = m.embed[first], torch.zeros(B, dtype=torch.int32, device=cuda)
    for layer in range(L):
        q, k, v = (heads(x @ w[layer], n) for w, n in ((m.wq, H), (m.wk, HKV), (m.wv, HKV)))
        rq, rk = rot(q, k)
        rq2 = append_paged(k, v, *pools[layer], table, none, prompt, rotary=rot, q=q)
        assert torch.equal(rq, rq2)
        o = flash_attention(rq, rk, v, causal=True)
        o = o[0] if isinstance(o, tuple) else o
        x = x + o.transpose(1, 2).reshape(B, most, H * D) @ m.wo[layer]
    x = x[torch.arange(B, device=cuda), prompt.long() - 1][:, None]
    lengths, tokens, logits = prompt, [], []
    for step in range(-1, STEPS):
        evicted(table, step)
        if step >= 0:
            seen, x = lengths + 1, m.embed[tokens[-1]][:, None]
            for layer in range(L):
                q, k, v = (heads(x @ w[layer], n) for w, n in ((m.wq, H), (m.wk, HKV), (m.wv, HKV)))
                q = append_paged(k, v, *pools[layer], table, lengths, rotary=rot, q=q)
                o = paged_attention(q, *pools[layer], table, seen)
                x = x + o.transpose(1, 2).reshape(B, 1, H * D) @ m.wo[layer]
            lengths = seen
        z = adjust_logits((x @ m.embed.T) * 0.1, history, lengths, prompt, repetition=repetition, presence=presence)
        _, _, token = verify_drafts(z, torch.zeros((B, 1), dtype=torch.int64, device=cuda), root, ones,
                                    m.noise[step + 1], temperature=temperature)
        history.scatter_(1, lengths.long()[:, None], token.int()[:, None])
        tokens.append(token)
        logits.append(z[:, 0])
    return torch.stack(tokens).cpu().numpy(), torch.stack(logits).double().cpu().numpy()


@pytest.mark.parametrize("interleaved, scaling", [(False, None), (True, dict(type="yarn", factor=4.0, original_length=16))])
def test_a_loop_of_steps(cuda, interleaved, scaling):
    rot = Rotary(D, rotary_dim=48, interleaved=interleaved, scaling=scaling).to(cuda)
    m = Model(3)
    table = np.random.default_rng(1).permutation(PAGES)[:B * COLUMNS].reshape(B, COLUMNS)
    want_tokens, want = oracle_loop(m.to(lambda t: t.double().numpy()), rot, 1.2, 0.3, 0.8, table)
    got_tokens, got = kernel_loop(m.to(lambda t: t.to(cuda)), rot, 1.2, 0.3, 0.8, table, cuda)
    np.testing.assert_array_equal(got_tokens, want_tokens)
    # fp32 throughout: two layers of sums of 256 terms of up to 10, logits of sums of 256 of up to 50
    # times 0.1; each sum is off by at most 256 * 2^-24 of its terms' size, the layers' errors add up.
    np.testing.assert_allclose(got, want, atol=256 * 2.0 ** -24 * 50, rtol=0)


def test_a_captured_step(cuda):
    """One step of two layers, replayed with other inputs, lengths and tables, eager work between."""
    rot = Rotary(D).to(cuda)
    g = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=g).bfloat16().to(cuda)
    pools = [[rand(PAGES, HKV, S, D) for _ in range(2)] for _ in range(L)]
    table = torch.randperm(PAGES, generator=g)[:B * COLUMNS].view(B, COLUMNS).int().to(cuda)
    lengths = torch.tensor([5, 0, 70], dtype=torch.int32, device=cuda)
    history = torch.randint(0, V, (B, COLUMNS * S), generator=g).int().to(cuda)
    q, k, v = rand(L, B, H, 1, D), rand(L, B, HKV, 1, D), rand(L, B, HKV, 1, D)
    logits, noise = rand(B, 1, V), torch.empty(B, V).exponential_(generator=g).to(cuda)
    last, root = torch.zeros((B, 1), dtype=torch.int64, device=cuda), torch.tensor([-1], dtype=torch.int32, device=cuda)
    ones = torch.zeros((B, 1), device=cuda)

    def step():
        seen = lengths + 1
        outs = []
        for i in range(L):
            turned = append_paged(k[i], v[i], *pools[i], table, lengths, rotary=rot, q=q[i])
            outs += paged_attention(turned, *pools[i], table, seen, return_lse=True)
        z = adjust_logits(logits, history, seen, repetition=1.3, frequency=0.1)
        _, _, token = verify_drafts(z, last, root, ones, noise, temperature=0.7)
        lengths.copy_(seen)
        return outs + [z, token]

    start = [x.clone() for pair in pools for x in pair], lengths.clone()
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for n in range(5):
        for x, y in zip((x for pair in pools for x in pair), start[0]):
            x.copy_(y)
        lengths.copy_(start[1] + 11 * n)
        for x in (q, k, v, logits):
            x.copy_(torch.randn(x.shape, generator=g))
        table[1, n] = -1
        want_at = lengths.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured] + [x.clone() for pair in pools for x in pair] + [lengths.clone()]
        for x, y in zip((x for pair in pools for x in pair), start[0]):
            x.copy_(y)
        lengths.copy_(want_at)
        want = step() + [x for pair in pools for x in pair] + [lengths]
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_two_streams_at_once(cuda):
    """Two requests' calls on streams of their own, with workspaces of their own."""
    rot = Rotary(D).to(cuda)
    g = torch.Generator().manual_seed(6)
    rand = lambda *s: torch.randn(s, generator=g).half().to(cuda)
    jobs = []
    for n in (700, 900):
        pages = -(-n // S) + 1
        jobs.append(dict(q=rand(1, H, 1, D), k=rand(pages, HKV, S, D), v=rand(pages, HKV, S, D),
                         table=torch.randperm(pages, generator=g).view(1, -1).int().to(cuda),
                         n=torch.tensor([n], dtype=torch.int32, device=cuda), x=rand(2, 1, 3001),
                         h=torch.randint(0, 3001, (2, 999), generator=g).int().to(cuda)))

    def work(j):
        out = paged_attention(rot(j["q"]), j["k"], j["v"], j["table"], j["n"], return_lse=True)
        return [*out, adjust_logits(j["x"], j["h"], presence=0.4, frequency=0.1)]

    want = [work(j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(20):
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(work(j))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for x, y in zip(outs, want[i % 2]):
            assert torch.equal(x, y)
