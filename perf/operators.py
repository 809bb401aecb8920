"""Speculative decoding over the K/V caches, as timed cases.

Each case names one operator with its sizes, data type and options:

  tree    tree_attention: a tree of drafted tokens (or one token a sequence) over caches whose
          sequences have lengths of their own
  verify  verify_drafts: the drafted tokens against the target's logits, from given random numbers
  cache   a model pass's drafted K and V appended to every layer's cache (append_drafts), then the
          accepted rows kept and the rest dropped (commit_drafts)

``listed()`` is the fixed set, ``draw()`` one more case of the same ranges. ``run()`` computes them
in plain torch, or with ``own`` by the framework's operators.
"""

from __future__ import annotations

import math
import pathlib
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
DEV = "cuda"
PACKAGE = "bridge-aware-kv-cache-eviction-for-efficient-long-context-transformers_amd"


def framework(module):
    """The framework's ``module``, from the repository in the working folder."""
    path = str(pathlib.Path.cwd() / PACKAGE)
    if path not in sys.path:
        sys.path.insert(0, path)
    return __import__("cab_attention." + module, fromlist=["*"])


def listed():
    return [
        # One request of a few hundred tokens with a short chain of drafts: all latency.
        dict(name="tree_chain_600", kind="tree", B=1, H=32, Hkv=8, T=5, N=600, D=128, dtype="bf16",
             shape="chain", ragged=False),
        # One request, a full tree over a cache of the evicting caches' usual size.
        dict(name="tree_64_8k", kind="tree", B=1, H=32, Hkv=8, T=64, N=8192, D=128, dtype="bf16",
             shape="tree", ragged=False),
        # A batch in the middle of serving: lengths and trees of their own, seven heads a group.
        dict(name="tree_ragged_16k", kind="tree", B=8, H=28, Hkv=4, T=26, N=16300, D=128,
             dtype="fp16", shape="tree", ragged=True),
        # fp32, head dim 64, a head of K and V for every query head, odd sizes.
        dict(name="tree_fp32_5k", kind="tree", B=2, H=12, Hkv=12, T=17, N=5003, D=64, dtype="fp32",
             shape="tree", ragged=True),
        # A batch without drafts: one token a sequence, lengths of their own.
        dict(name="token_batch_32k", kind="tree", B=16, H=32, Hkv=8, T=1, N=32768, D=128,
             dtype="bf16", shape="chain", ragged=True),
        # Long contexts with full trees: the largest.
        dict(name="tree_batch_64k", kind="tree", B=4, H=32, Hkv=8, T=64, N=65536, D=128,
             dtype="bf16", shape="tree", ragged=True),
        # Greedy decoding with a chain of four drafts.
        dict(name="verify_greedy", kind="verify", B=1, T=5, V=32000, dtype="fp16", mode="greedy",
             temperature=0.0, shape="chain"),
        # Sampling, a full tree of the draft's most likely tokens, a large vocabulary.
        dict(name="verify_tree", kind="verify", B=1, T=64, V=128000, dtype="bf16", mode="point",
             temperature=0.8, shape="tree"),
        # Sampling against the draft model's own distribution, odd vocabulary, fp32 logits.
        dict(name="verify_drafted", kind="verify", B=4, T=26, V=50001, dtype="fp32", mode="draft",
             temperature=1.0, shape="tree"),
        # A serving batch's trees in one call.
        dict(name="verify_batch", kind="verify", B=32, T=32, V=128000, dtype="bf16", mode="point",
             temperature=1.0, shape="tree"),
        # One request's chain through a whole model's caches.
        dict(name="cache_chain", kind="cache", L=28, B=1, H=4, T=5, N=2000, D=128, dtype="bf16",
             shape="chain", keep=3),
        # A batch's trees through a whole model's caches.
        dict(name="cache_batch", kind="cache", L=32, B=4, H=8, T=64, N=1500, D=128, dtype="bf16",
             shape="tree", keep=6),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "verify", "verify", "cache"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    shape = rng.choice(["tree", "tree", "chain"])
    if kind == "tree":
        c = dict(kind=kind, Hkv=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128]), dtype=dtype,
                 T=spread(rng, 1, 128), shape=shape, ragged=rng.random() < 0.7)
        c["H"] = c["Hkv"] * rng.choice([1, 2, 3, 4, 5, 7, 8])
        c["B"] = spread(rng, 1, 16)
        # At most a third of the largest listed case's work, and an eighth of that in fp32.
        most = (1 << 34) // (8 if dtype == "fp32" else 1) // (c["B"] * c["H"] * c["D"] * c["T"])
        room = (1 << 29) // (c["B"] * c["Hkv"] * c["D"] * 2 * BYTES[dtype])
        c["N"] = c["T"] + spread(rng, 1, max(2, min(65536, most, room)))
        return c
    if kind == "verify":
        c = dict(kind=kind, V=spread(rng, 1000, 150000), dtype=dtype, shape=shape,
                 mode=rng.choice(["greedy", "point", "point", "draft"]), T=spread(rng, 1, 64))
        c["temperature"] = 0.0 if c["mode"] == "greedy" else round(rng.uniform(0.4, 1.3), 2)
        most = (1 << 27) // (c["V"] * c["T"] * (2 if c["mode"] == "draft" else 1))
        c["B"] = spread(rng, 1, max(1, min(32, most)))
        return c
    c = dict(kind=kind, L=rng.randint(1, 32), H=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128]),
             T=spread(rng, 1, 64), B=spread(rng, 1, 4), dtype=rng.choice(["bf16", "fp16", "fp32"]),
             shape=shape)
    c["N"] = c["T"] + spread(rng, 100, 1500)
    c["keep"] = rng.randint(1, min(8, c["T"]))
    return c


def trees(case, seed):
    """Parents ``[B, T]``: node 0 is the root; a node hangs on any earlier one, or on the one before
    (a chain). In a ragged batch the last nodes of some sequences are absent (-2)."""
    rng = random.Random(seed)
    T = case["T"]
    rows = []
    for b in range(case["B"]):
        n = rng.randint(max(1, T - 6), T) if case.get("ragged") and case["shape"] == "tree" else T
        rows.append([-1 if i == 0 else -2 if i >= n else
                     i - 1 if case["shape"] == "chain" else int(i * rng.random())
                     for i in range(T)])
    return torch.tensor(rows, dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed + 1)
    parents = trees(case, seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case, parents=parents.to(DEV))
    if case["kind"] == "tree":
        B, H, Hkv, T, N, D = (case[x] for x in ("B", "H", "Hkv", "T", "N", "D"))
        most = N - T
        lengths = [rng.randint(most // 4, most) if case["ragged"] else most for _ in range(B)]
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        # As a projection leaves them: [B, T, H, D]; the cache is [B, H_kv, N, D]. Queries
        # somewhat longer than unit variance, so that attention is not flat.
        s["q"] = (1.5 * torch.randn((B, T, H, D), generator=g, device=DEV)).to(dt).transpose(1, 2)
        s["k"] = torch.randn((B, Hkv, N, D), generator=g, device=DEV).to(dt)
        s["v"] = torch.randn((B, Hkv, N, D), generator=g, device=DEV).to(dt)
        return s
    if case["kind"] == "verify":
        B, T, V = case["B"], case["T"], case["V"]
        # A few likely tokens stand out of each row; the vocabulary's padding is masked.
        top = torch.randint(0, V - V // 500 - 1, (B, T, 6), generator=g, device=DEV)
        lift = (7.0 + 5.0 * torch.rand((B, T, 6), generator=g, device=DEV)).sort(2, True).values
        logits = torch.empty((B, T, V), dtype=dt, device=DEV)
        drafts = torch.empty_like(logits) if case["mode"] == "draft" else None
        par = parents.to(DEV, torch.int64).clamp(min=0)
        tokens = torch.empty((B, T), dtype=torch.int64, device=DEV)
        # A node's children in turn: its likeliest token, the next one, ...
        pick = torch.tensor([[min(5, up[:i].count(up[i])) for i in range(T)]
                             for up in parents.tolist()], device=DEV)
        for b in range(B):
            x = torch.randn((T, V), generator=g, device=DEV).scatter_(1, top[b], lift[b])
            x[:, V - V // 500:] = -math.inf
            logits[b] = x.to(dt)
            tokens[b] = top[b][par[b], pick[b]]
            if drafts is not None:
                # The draft's logits are the target's with an error; its tokens a sample of them.
                drafts[b] = (x + 0.7 * torch.randn((T, V), generator=g, device=DEV)).to(dt)
                e = torch.empty((T, V), device=DEV).exponential_(generator=g)
                tokens[b] = (drafts[b].float()[par[b]] / case["temperature"] - e.log()).argmax(1)
        if case["mode"] == "greedy":
            # Four drafts in five are the target's own choice.
            best = logits.float().argmax(2).gather(1, par)
            hit = torch.rand((B, T), generator=g, device=DEV) < 0.8
            tokens = torch.where(hit, best, tokens)
        s.update(logits=logits, drafts=drafts, tokens=tokens)
        s["uniforms"] = torch.rand((B, T), generator=g, device=DEV)
        s["noise"] = torch.empty((B, V), device=DEV).exponential_(generator=g)
        return s
    L, B, H, T, N, D = (case[x] for x in ("L", "B", "H", "T", "N", "D"))
    # Every layer's K and V, and the drafted rows as the projections leave them.
    s["buffers"] = torch.randn((2 * L, B, H, N, D), generator=g, device=DEV, dtype=torch.float32).to(dt)
    s["new"] = torch.randn((2 * L, B, T, H, D), generator=g, device=DEV).to(dt).transpose(2, 3)
    s["caches"] = list(s["buffers"].unbind(0))
    s["lengths"] = torch.tensor([rng.randint((N - T) // 2, N - T) for _ in range(B)],
                                dtype=torch.int32, device=DEV)
    # An accepted path: up to ``keep`` nodes from the root down.
    paths, counts = [], []
    for b in range(B):
        path, want = [0], rng.randint(1, case["keep"])
        up = parents[b].tolist()
        while len(path) < want:
            below = [i for i in range(T) if up[i] == path[-1]]
            if not below:
                break
            path.append(rng.choice(below))
        counts.append(len(path))
        paths.append(path + [-1] * (T - len(path)))
    s["path"] = torch.tensor(paths, dtype=torch.int32, device=DEV)
    s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def ancestors(parents):
    """``seen[b, i, j]``: whether j is i or one of its ancestors; a node that is absent or hangs on
    an absent one sees nothing."""
    B, T = parents.shape
    p = parents.long()
    i = torch.arange(T, device=p.device)
    linked = (p >= 0) & (p < i)
    present = linked | (p == -1)
    up = torch.where(linked, p, i)  # a root, and an absent node, stays where it is
    seen = torch.eye(T, dtype=torch.bool, device=p.device).expand(B, T, T)
    for _ in range(max(1, (T - 1).bit_length())):  # twice the distance each time
        seen = seen | seen.gather(1, up[:, :, None].expand(B, T, T))
        present = present & present.gather(1, up)
        up = up.gather(1, up)
    return seen & present[:, :, None]


def plain_tree(s):
    q, k, v, lengths = s["q"].float(), s["k"].float(), s["v"].float(), s["lengths"].long()
    B, H, T, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    j = torch.arange(N, device=q.device)[None, :] - lengths[:, None]  # key's node, < 0: context
    seen = ancestors(s["parents"])
    some = seen.any(2)
    mask = torch.where((j < 0)[:, None, :], some[:, :, None],
                       seen.gather(2, j.clamp(0, T - 1)[:, None, :].expand(B, T, N))
                       & (j < T)[:, None, :])
    score = torch.matmul(q.reshape(B, Hkv, H // Hkv * T, D), k.transpose(2, 3)) / math.sqrt(D)
    score = score.reshape(B, Hkv, H // Hkv, T, N).masked_fill(~mask[:, None, None], -math.inf)
    high = score.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(score - high)
    total = e.sum(-1, keepdim=True)
    v = torch.where((j < T)[:, None, :, None], v, 0.0)  # (rows behind a sequence hold anything)
    out = torch.matmul((e / total.clamp(min=1e-30)).reshape(B, Hkv, -1, N), v)
    lse = (high + torch.log(total))[..., 0].reshape(B, H, T)
    return [out.reshape(B, H, T, D).to(s["q"].dtype), lse]


def weights(logits, temperature):
    """softmax(logits / temperature) in 64 bits: every sum here meets a border."""
    x = logits.double() / temperature
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def plain_verify(s):
    case, logits, drafts = s["case"], s["logits"], s["drafts"]
    tokens, parents, uniforms = s["tokens"], s["parents"], s["uniforms"].double()
    B, T, V = logits.shape
    mode, temperature = case["mode"], case["temperature"]
    rows = torch.arange(B, device=logits.device)
    at = torch.zeros(B, dtype=torch.long, device=logits.device)
    took = torch.zeros((B, T), dtype=torch.bool, device=logits.device)
    took[:, 0] = True
    # w: what is left of the target's weights at each sequence's node, c its sum, a: see below.
    p = w = q = a = None
    if mode != "greedy":
        p = w = weights(logits[:, 0], temperature)
        c, a = w.sum(1), torch.zeros(B, dtype=torch.float64, device=logits.device)
    if mode == "draft":
        q = weights(drafts[:, 0], temperature)
    for i in range(1, T):
        child = parents[:, i] == at
        x = tokens[:, i]
        if mode == "greedy":
            took[:, i] = child & (logits[rows, at].float().argmax(1) == x)
        else:
            left = w.gather(1, x[:, None])[:, 0]
            of = q.gather(1, x[:, None])[:, 0] if mode == "draft" else 1.0
            took[:, i] = child & (uniforms[:, i] * c * of < left)
            out = child & ~took[:, i]
            if mode == "draft":
                # max(max(p - a q, 0) / c - q, 0) is max(p - (a + c) q, 0) / c
                a = torch.where(out, a + c, a)
                w = (p - a[:, None] * q).clamp(min=0)
            else:
                w = w.scatter(1, x[:, None], torch.where(out, 0.0, left)[:, None])
            new = took[:, i, None]
            p = torch.where(new, weights(logits[:, i], temperature), p)
            w = torch.where(new, p, w)
            if mode == "draft":
                q = torch.where(new, weights(drafts[:, i], temperature), q)
                a = torch.where(took[:, i], 0.0, a)
            c = w.sum(1)
        at = torch.where(took[:, i], i, at)
    if mode == "greedy":
        token = logits[rows, at].float().argmax(1)
    else:
        token = (torch.where((c > 0)[:, None], w, p) / s["noise"].double()).argmax(1)
    counts = took.sum(1)
    node = torch.where(took, torch.arange(T, device=logits.device), T).sort(1).values
    return [torch.where(node < T, node, -1).int(), counts.int(), token]


def plain_cache(s):
    case, buffers, new = s["case"], s["buffers"], s["new"]
    L, B, T = case["L"], case["B"], case["T"]
    rows = s["lengths"].long()[:, None] + torch.arange(T, device=buffers.device)
    batch = torch.arange(B, device=buffers.device)[:, None]
    for layer in range(L):  # a layer's K and V are there when the layer has run
        buffers[2 * layer][batch, :, rows] = new[2 * layer].transpose(1, 2)
        buffers[2 * layer + 1][batch, :, rows] = new[2 * layer + 1].transpose(1, 2)
    kept = torch.arange(T, device=buffers.device) < s["counts"][:, None]
    source = torch.where(kept, s["lengths"][:, None] + s["path"], rows).long()
    moved = buffers.transpose(2, 3)[:, batch, source]
    buffers.transpose(2, 3)[:, batch, rows] = moved
    return [s["lengths"] + s["counts"], buffers]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"tree": plain_tree, "verify": plain_verify, "cache": plain_cache}[kind](state)
    if kind == "tree":
        return list(framework("kernels").tree_attention(
            state["q"], state["k"], state["v"], state["parents"], state["lengths"],
            return_lse=True))
    if kind == "verify":
        return list(framework("kernels").verify_drafts(
            state["logits"], state["tokens"], state["parents"], state["uniforms"], state["noise"],
            temperature=state["case"]["temperature"], draft_logits=state["drafts"]))
    cache, new, caches = framework("cache"), state["new"], state["caches"]
    for layer in range(state["case"]["L"]):
        cache.append_drafts(new[2 * layer], new[2 * layer + 1], caches[2 * layer],
                            caches[2 * layer + 1], state["lengths"])
    return [cache.commit_drafts(caches, state["lengths"], state["path"], state["counts"]),
            state["buffers"]]


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its value in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "tree":
        B, H, Hkv, T, D = (case[x] for x in ("B", "H", "Hkv", "T", "D"))
        keys = (case["N"] - T) * (0.625 if case["ragged"] else 1.0) + T  # of a sequence, on average
        return {"bytes": 2 * B * Hkv * keys * D * e + 2 * B * H * T * D * e + 4 * B * H * T,
                "flops": 4 * B * H * T * keys * D}
    if case["kind"] == "verify":
        # The rows of the accepted nodes: the root's and about two more (a chain of 20 greedy
        # drafts, accepted at four in five: about four).
        rows = min(case["T"], 5 if case["mode"] == "greedy" else 3)
        V, B = case["V"], case["B"]
        read = rows * V * e * (2 if case["mode"] == "draft" else 1)
        return {"bytes": B * (read + (0 if case["mode"] == "greedy" else 4 * V)),
                "flops": B * rows * V * (1 if case["mode"] == "greedy" else 4)}
    rows = case["T"] + (case["keep"] + 1) / 2
    return {"bytes": 4 * case["L"] * case["B"] * case["H"] * rows * case["D"] * e, "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "cache":
        T, buffers = case["T"], s["buffers"].double()
        for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
            buffers[:, b, :, n:n + T] = s["new"][:, b].double()
            kept = [n + x for x in s["path"][b].tolist()[:c]]
            buffers[:, b, :, n:n + c] = buffers[:, b, :, kept].clone()
        return [s["lengths"] + s["counts"], buffers]
    if case["kind"] == "tree":
        out, lse = [], []
        group = case["H"] // case["Hkv"]
        for b in range(case["B"]):
            n = int(s["lengths"][b])
            up = s["parents"][b].tolist()
            seen = torch.zeros((case["T"], n + case["T"]), dtype=torch.bool, device=DEV)
            for i in range(case["T"]):
                j, line = i, []
                while 0 <= j and 0 <= up[j] < j:
                    line.append(j)
                    j = up[j]
                if up[j] == -1:
                    seen[i, :n] = True
                    seen[i, torch.tensor([n + x for x in line + [j]], device=DEV)] = True
            rows, sums = [], []
            for h in range(case["H"]):
                k, v = (s[x][b, h // group, :n + case["T"]].double() for x in "kv")
                z = (s["q"][b, h].double() @ k.T) * case["D"] ** -0.5
                z = torch.where(seen, z, -math.inf)
                total = torch.logsumexp(z, 1)
                weight = torch.where(seen, torch.exp(z - total.clamp(min=-1e300)[:, None]), 0.0)
                rows.append(weight @ v)
                sums.append(total)
            out.append(torch.stack(rows))
            lse.append(torch.stack(sums))
        return [torch.stack(out), torch.stack(lse)]
    paths, counts, chosen = [], [], []
    t = case["temperature"]
    for b in range(case["B"]):
        up, tokens = s["parents"][b].tolist(), s["tokens"][b].tolist()
        r = s["uniforms"][b].double().tolist()
        path = [0]
        while True:
            node, step = path[-1], None
            row = s["logits"][b, node].double()
            left = torch.softmax(row / t, 0) if t else None
            other = torch.softmax(s["drafts"][b, node].double() / t, 0) if case["mode"] == "draft" else None
            for i in [i for i in range(case["T"]) if up[i] == node]:
                x = tokens[i]
                if case["mode"] == "greedy":
                    ok = x == int((row == row.max()).nonzero()[0])
                elif case["mode"] == "point":
                    ok = r[i] < float(left[x])
                else:
                    ok = r[i] * float(other[x]) < float(left[x])
                if ok:
                    step = i
                    break
                if case["mode"] == "point":
                    left = left.clone()
                    left[x] = 0.0
                    left = left / left.sum()
                elif case["mode"] == "draft":
                    left = (left - other).clamp(min=0)
                    left = left / left.sum()
            if step is None:
                break
            path.append(step)
        best = row if not t else left / s["noise"][b].double()
        chosen.append(int((best == best.max()).nonzero()[0]))
        counts.append(len(path))
        paths.append(path + [-1] * (case["T"] - len(path)))
    return [torch.tensor(paths), torch.tensor(counts), torch.tensor(chosen)]
