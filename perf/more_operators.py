"""Decoding over a paged K/V cache with rotary positions, as timed cases.

Each case names one operator with its sizes, data type and options:

  rotate  Rotary: rotary positions on a prompt's queries and keys, in training with its gradient
  append  append_paged: a model pass's new K and V into every layer's pages, K and the queries
          rotated to their positions on the way
  attend  paged_attention: one token of every sequence over the pages of its cache
  adjust  adjust_logits: penalties for repeated tokens, biases and grammar masks, for one token a
          sequence or for a tree of drafts

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
TRAINED = 4096  # the context that scaled frequencies start from


def framework(module):
    """The framework's ``module``, from the repository in the working folder."""
    path = str(pathlib.Path.cwd() / PACKAGE)
    if path not in sys.path:
        sys.path.insert(0, path)
    return __import__("cab_attention." + module, fromlist=["*"])


def listed():
    return [
        # A self-attention module's queries and keys, a part of each head in interleaved pairs.
        dict(name="rotate_module", kind="rotate", B=2, H=8, Hkv=8, N=4096, D=64, R=32, dtype="fp32",
             interleaved=True, scaling="none", factor=1.0, train=False, ragged=False),
        # A long prompt past the trained context.
        dict(name="rotate_prompt_16k", kind="rotate", B=1, H=32, Hkv=8, N=16384, D=128, R=128,
             dtype="bf16", interleaved=False, scaling="yarn", factor=4.0, train=False, ragged=False),
        # Training on packed documents (positions of their own), forward and backward.
        dict(name="rotate_train", kind="rotate", B=2, H=28, Hkv=4, N=16300, D=128, R=128,
             dtype="fp16", interleaved=False, scaling="linear", factor=4.0, train=True, ragged=True),
        # One token of a small batch through a whole model: launches count.
        dict(name="append_tokens", kind="append", L=28, B=16, H=28, Hkv=4, T=1, N=256, S=16, D=128,
             R=128, dtype="bf16", interleaved=False, scaling="yarn", factor=4.0),
        # A chunk of several prompts through a few layers, counts of their own, half of each head.
        dict(name="append_prompts", kind="append", L=4, B=4, H=32, Hkv=8, T=2000, N=4096, S=64,
             D=128, R=64, dtype="fp16", interleaved=True, scaling="none", factor=1.0),
        # One request of a few hundred tokens: all latency.
        dict(name="attend_600", kind="attend", B=1, H=32, Hkv=8, N=600, S=16, D=128, dtype="bf16",
             ragged=False, dropped=0.0),
        # fp32, pages of an odd size, a head of K and V for every query head, a quarter of the
        # pages evicted.
        dict(name="attend_fp32_5k", kind="attend", B=3, H=12, Hkv=12, N=5003, S=24, D=64,
             dtype="fp32", ragged=True, dropped=0.25),
        # One request with a long context: its keys have to be spread over the chip.
        dict(name="attend_long", kind="attend", B=1, H=28, Hkv=4, N=128000, S=64, D=128,
             dtype="fp16", ragged=False, dropped=0.0),
        # A serving batch with lengths of their own: the largest.
        dict(name="attend_batch_32k", kind="attend", B=16, H=32, Hkv=8, N=32768, S=16, D=128,
             dtype="bf16", ragged=True, dropped=0.0),
        # One request's next token: penalties and a few biases.
        dict(name="adjust_one", kind="adjust", B=1, T=1, V=32000, L=600, dtype="fp16", biases=10,
             masked=False, shape="chain"),
        # Trees of drafts under a grammar, odd vocabulary.
        dict(name="adjust_trees", kind="adjust", B=4, T=26, V=50001, L=5003, dtype="fp32",
             biases=0, masked=True, shape="tree"),
        # A serving batch with long histories, a large vocabulary, everything at once.
        dict(name="adjust_batch", kind="adjust", B=64, T=1, V=128000, L=8192, dtype="bf16",
             biases=100, masked=True, shape="chain"),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "attend", "attend", "adjust"])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if kind == "adjust":
        c.update(T=rng.choice([1, 1, spread(rng, 2, 48)]), V=spread(rng, 1000, 150000),
                 L=spread(rng, 1, 16384), biases=rng.choice([0, spread(rng, 1, 300)]),
                 masked=rng.random() < 0.6, shape=rng.choice(["tree", "chain"]))
        c["B"] = spread(rng, 1, max(1, min(64, (1 << 22) // (c["T"] * c["V"]))))
        return c
    c.update(Hkv=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128]))
    c["H"] = c["Hkv"] * rng.choice([1, 2, 3, 4, 5, 7, 8])
    if kind == "attend":
        c.update(B=spread(rng, 1, 32), S=rng.choice([8, 16, 16, 20, 32, 64, 128, 256]),
                 ragged=rng.random() < 0.7, dropped=rng.choice([0.0, 0.0, 0.3]))
        room = (1 << 29) // (c["B"] * c["Hkv"] * c["D"] * 2 * BYTES[c["dtype"]])
        c["N"] = spread(rng, 1, max(2, min(131072, room)))
        return c
    c.update(R=rng.choice([c["D"], c["D"], c["D"] // 2, 16]), interleaved=rng.random() < 0.4,
             scaling=rng.choice(["none", "linear", "yarn"]))
    c["factor"] = 1.0 if c["scaling"] == "none" else rng.choice([2.0, 4.0, 7.5])
    width = (c["H"] + c["Hkv"]) * c["D"] * BYTES[c["dtype"]]
    if kind == "rotate":
        c.update(B=spread(rng, 1, 8), train=rng.random() < 0.5, ragged=rng.random() < 0.5)
        c["N"] = spread(rng, 1, max(2, min(32768, (1 << 27) // (c["B"] * width))))
        return c
    c.update(L=rng.randint(1, 28), B=spread(rng, 1, 16), S=rng.choice([8, 16, 20, 32, 64]))
    c["T"] = spread(rng, 1, max(2, min(2048, (1 << 28) // (c["L"] * c["B"] * width))))
    c["N"] = c["T"] + spread(rng, 32, 256)
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def frequencies(case):
    """Radians a position for each pair ``[R / 2]`` (64 bits), and the amplitude."""
    R, base, factor = case["R"], 10000.0, case["factor"]
    i = torch.arange(R // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / R)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        # Pairs that turn more than 32 times within the trained context stay, those that turn
        # less than once are stretched, a ramp between them.
        low, high = (R * math.log(TRAINED / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32, 1))
        low, high = max(math.floor(low), 0), min(math.ceil(high), R - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def rotary(case):
    """The framework's module, as a model keeps it."""
    scaling = None if case["scaling"] == "none" else {"type": case["scaling"], "factor": case["factor"]}
    if case["scaling"] == "yarn":
        scaling["original_length"] = TRAINED
    return framework("kernels").Rotary(case["D"], rotary_dim=case["R"], scaling=scaling,
                                       interleaved=case["interleaved"]).to(DEV)


def page_table(rng, lengths, columns, size, dropped=0.0):
    """Pages in the order in which a server that has run for a while hands them out: any. A table
    ``[B, columns]`` (-1: no page), and how many pages there are."""
    need = [-(-n // size) for n in lengths]
    pages = len(need) * columns + 3  # room for every sequence at its longest
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(rng.randrange(1 << 30)))
    table = torch.full((len(need), columns), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = free[at:at + n].int()
        at += n
        for i in rng.sample(range(max(0, n - 1)), int(dropped * max(0, n - 1))):
            table[b, i] = -1  # evicted; a sequence's last page stays
    return table, pages


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed + 1)
    dt, kind, B = DTYPES[case["dtype"]], case["kind"], case["B"]
    s = dict(case=case)

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(shape, generator=g, device=DEV)).to(dt)

    if kind == "rotate":
        H, Hkv, N, D = (case[x] for x in ("H", "Hkv", "N", "D"))
        # As a projection leaves them: [B, N, H, D].
        s["q"], s["k"] = normal(B, N, H, D).transpose(1, 2), normal(B, N, Hkv, D).transpose(1, 2)
        if case["train"]:
            s["gq"], s["gk"] = normal(B, N, H, D).transpose(1, 2), normal(B, N, Hkv, D).transpose(1, 2)
        s["positions"] = None
        if case["ragged"]:  # two documents in each row
            cut = torch.tensor([[rng.randint(0, N)] for _ in range(B)])
            at = torch.arange(N).expand(B, N)
            s["positions"] = torch.where(at < cut, at, at - cut).int().to(DEV)
        s["frequencies"], s["amplitude"] = frequencies(case)
        if own:
            s["rotary"] = rotary(case)
        return s
    if kind == "append":
        L, H, Hkv, T, N, S, D = (case[x] for x in ("L", "H", "Hkv", "T", "N", "S", "D"))
        lengths = [rng.randint(0, N - T) for _ in range(B)]
        table, pages = page_table(rng, [n + T for n in lengths], -(-N // S), S)
        s["table"] = table.to(DEV)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        counts = [rng.randint(max(1, T // 2), T) for _ in range(B)]
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
        s["pages"] = torch.empty((2 * L, pages, Hkv, S, D), dtype=dt, device=DEV)
        for x in s["pages"]:
            x.copy_(normal(pages, Hkv, S, D))
        s["q"] = normal(L, B, T, H, D).transpose(2, 3)
        s["new"] = normal(2 * L, B, T, Hkv, D).transpose(2, 3)
        s["frequencies"], s["amplitude"] = frequencies(case)
        if own:
            s["rotary"] = rotary(case)
        return s
    if kind == "attend":
        H, Hkv, N, S, D = (case[x] for x in ("H", "Hkv", "N", "S", "D"))
        lengths = [rng.randint(max(1, N // 4), N) if case["ragged"] else N for _ in range(B)]
        table, pages = page_table(rng, lengths, -(-N // S), S, case["dropped"])
        s["table"] = table.to(DEV)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        # Queries somewhat longer than unit variance, so that attention is not flat.
        s["q"] = normal(B, 1, H, D, scale=1.5).transpose(1, 2)
        s["k"], s["v"] = normal(pages, Hkv, S, D), normal(pages, Hkv, S, D)
        return s
    T, V, L = case["T"], case["V"], case["L"]
    # Logits as a model gives them: a few tokens stand out, the repeated ones among them.
    # Text repeats itself: tokens by a power law over the vocabulary.
    rank = torch.rand((B, L + T), generator=g, device=DEV).pow(4)
    words = (rank * V).long().clamp(max=V - 1)
    s["history"] = words[:, :L].int().contiguous()
    s["drafts"] = words[:, L:].contiguous() if T > 1 else None
    lengths = [rng.randint(L // 2, L) for _ in range(B)]
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    s["prompts"] = torch.tensor([rng.randint(0, n) for n in lengths], dtype=torch.int32, device=DEV)
    parents = [[-1 if i == 0 else i - 1 if case["shape"] == "chain" else int(i * rng.random())
                for i in range(T)] for _ in range(B)]
    s["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV) if T > 1 else None
    s["logits"] = normal(B, T, V, scale=3.0)
    # Each request has penalties of its own.
    s["repetition"] = 1.0 + 0.3 * torch.rand(B, generator=g, device=DEV)
    s["presence"] = 0.6 * torch.rand(B, generator=g, device=DEV)
    s["frequency"] = 0.2 * torch.rand(B, generator=g, device=DEV)
    s["bias_tokens"] = s["bias"] = s["allowed"] = None
    if case["biases"]:
        n = min(case["biases"], V)
        s["bias_tokens"] = torch.rand((B, V), generator=g, device=DEV).argsort(1)[:, :n].int().contiguous()
        s["bias"] = 4.0 * torch.randn((B, n), generator=g, device=DEV)
    if case["masked"]:
        # A grammar's state allows a tenth of the tokens, as bits.
        bits = torch.zeros((B, T, -(-V // 32) * 32), dtype=torch.bool, device=DEV)
        bits[:, :, :V] = torch.rand((B, T, V), generator=g, device=DEV) < 0.1
        value = bits.view(B, T, -1, 32).long() << torch.arange(32, device=DEV)
        word = value.sum(3)
        s["allowed"] = torch.where(word >= 1 << 31, word - (1 << 32), word).int()
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def rotated(x, positions, frequency, amplitude, interleaved, sign=1.0):
    """x ``[B, H, n, D]`` in 32 bits, turned by ``positions`` ``[B, n]``; angles in 64 bits."""
    half = frequency.numel()
    angle = positions.double()[:, None, :, None] * frequency.to(x.device)
    cos = (torch.cos(angle) * amplitude).float()
    sin = (torch.sin(angle) * (amplitude * sign)).float()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def plain_rotate(s):
    case, q, positions = s["case"], s["q"], s["positions"]
    if positions is None:
        positions = torch.arange(case["N"], device=q.device).expand(case["B"], -1)
    turn = lambda x, sign: rotated(x.float(), positions, s["frequencies"], s["amplitude"],
                                   case["interleaved"], sign).to(x.dtype)
    out = [turn(q, 1.0), turn(s["k"], 1.0)]
    if case["train"]:  # the transpose of a rotation turns back
        out += [turn(s["gq"], -1.0), turn(s["gk"], -1.0)]
    return out


def plain_append(s):
    case, pages, new, table = s["case"], s["pages"], s["new"], s["table"].long()
    B, T, S = case["B"], case["T"], case["S"]
    t = torch.arange(T, device=pages.device)
    positions = s["lengths"].long()[:, None] + t
    inside = (t < s["counts"][:, None]).nonzero(as_tuple=True)
    at = positions[inside]
    page, place = table[inside[0], at // S], at % S
    out = []
    for layer in range(case["L"]):  # a layer's K and V are there when the layer has run
        turn = lambda x: rotated(x.float(), positions, s["frequencies"], s["amplitude"],
                                 case["interleaved"]).to(x.dtype)
        out.append(turn(s["q"][layer]))
        pages[2 * layer][page, :, place] = turn(new[2 * layer]).transpose(1, 2)[inside]
        pages[2 * layer + 1][page, :, place] = new[2 * layer + 1].transpose(1, 2)[inside]
    return out + [pages]


def plain_attend(s):
    q, table, lengths = s["q"].float(), s["table"].long(), s["lengths"]
    B, H, _, D = q.shape
    _, Hkv, S, _ = s["k"].shape
    n = table.shape[1] * S
    gathered = lambda x: x[table.clamp(min=0)].transpose(1, 2).reshape(B, Hkv, n, D).float()
    there = (table >= 0)[:, :, None].expand(-1, -1, S).reshape(B, n)
    mask = (there & (torch.arange(n, device=q.device) < lengths[:, None]))[:, None]
    score = torch.matmul(q.reshape(B, Hkv, H // Hkv, D), gathered(s["k"]).transpose(2, 3)) / math.sqrt(D)
    score = score.masked_fill(~mask[:, None], -math.inf).reshape(B, H, n)
    high = score.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(score - high)
    total = e.sum(-1, keepdim=True)
    v = torch.where(mask[..., None], gathered(s["v"]), 0.0)  # (other places hold anything)
    out = torch.matmul((e / total.clamp(min=1e-30)).reshape(B, Hkv, -1, n), v)
    return [out.reshape(B, H, 1, D).to(s["q"].dtype), high + torch.log(total)]


def lines(parents):
    """``line[b, i, j]``: whether node j is i or one of its ancestors."""
    B, T = parents.shape
    i = torch.arange(T, device=parents.device)
    up = torch.where(parents >= 0, parents.long(), i)
    line = torch.eye(T, dtype=torch.bool, device=parents.device).expand(B, T, T)
    for _ in range(max(1, (T - 1).bit_length())):  # twice the distance each time
        line = line | line.gather(1, up[:, :, None].expand(B, T, T))
        up = up.gather(1, up)
    return line


def plain_adjust(s):
    logits = s["logits"]
    B, T, V = logits.shape
    x = logits.float()
    at = torch.arange(s["history"].shape[1], device=x.device)
    words = s["history"].long()
    given = at < s["prompts"][:, None]
    made = (at < s["lengths"][:, None]) & ~given
    tally = lambda what: torch.zeros((B, V), device=x.device).scatter_add_(1, words, what.float())
    prompt, count = tally(given) > 0, tally(made)[:, None]
    if s["drafts"] is not None:
        tokens = s["drafts"][:, None, :].expand(B, T, T)
        count = count.expand(B, T, V).scatter_add(2, tokens, lines(s["parents"]).float())
    seen = (count > 0) | prompt[:, None]
    r, p, f = (s[k][:, None, None] for k in ("repetition", "presence", "frequency"))
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - f * count - p * (count > 0)
    if s["bias"] is not None:
        dense = torch.zeros((B, V), device=x.device).scatter_(1, s["bias_tokens"].long(), s["bias"])
        x = x + dense[:, None]
    if s["allowed"] is not None:
        v = torch.arange(V, device=x.device)
        x = x.masked_fill((s["allowed"][..., v // 32] >> (v % 32)) & 1 == 0, -math.inf)
    return x.to(logits.dtype)


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"rotate": plain_rotate, "append": plain_append, "attend": plain_attend,
                "adjust": plain_adjust}[kind](state)
    if kind == "rotate":
        q, k = state["q"], state["k"]
        if not state["case"]["train"]:
            return list(state["rotary"](q, k, state["positions"]))
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = state["rotary"](q, k, state["positions"])
        return list(out) + list(torch.autograd.grad(out, (q, k), (state["gq"], state["gk"])))
    if kind == "append":
        cache, pages, new = framework("cache"), state["pages"], state["new"]
        out = [cache.append_paged(new[2 * layer], new[2 * layer + 1], pages[2 * layer],
                                  pages[2 * layer + 1], state["table"], state["lengths"],
                                  state["counts"], rotary=state["rotary"], q=state["q"][layer])
               for layer in range(state["case"]["L"])]
        return out + [pages]
    if kind == "attend":
        return list(framework("kernels").paged_attention(
            state["q"], state["k"], state["v"], state["table"], state["lengths"], return_lse=True))
    return framework("kernels").adjust_logits(
        state["logits"], state["history"], state["lengths"], state["prompts"],
        repetition=state["repetition"], presence=state["presence"], frequency=state["frequency"],
        bias_tokens=state["bias_tokens"], bias=state["bias"], allowed=state["allowed"],
        drafts=state["drafts"], parents=state["parents"])


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its value in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    e, kind, B, T = BYTES[case["dtype"]], case["kind"], case["B"], case.get("T", 1)
    if kind == "adjust":
        V = case["V"]
        read = 2 * B * T * V * e + 4 * B * case["L"] * 0.75 + 8 * B * case["biases"]
        return {"bytes": read + (B * T * V / 8 if case["masked"] else 0), "flops": B * T * V}
    H, Hkv, N, D = (case[x] for x in ("H", "Hkv", "N", "D"))
    if kind == "attend":
        keys = N * (0.625 if case["ragged"] else 1.0) * (1 - case["dropped"])  # on average
        return {"bytes": 2 * B * Hkv * keys * D * e + 2 * B * H * D * e + 4 * B * H,
                "flops": 4 * B * H * keys * D}
    turned = 3 * case["R"]  # two products and a sum a value
    if kind == "rotate":
        n = B * N * (H + Hkv) * (2 if case["train"] else 1)
        return {"bytes": 2 * n * D * e, "flops": n * turned}
    n, kept = case["L"] * B * T, case["L"] * B * (T + 1) * (0.75 if T > 1 else 0.5)
    return {"bytes": 2 * (n * H + 2 * kept * Hkv) * D * e, "flops": (n * H + kept * Hkv) * turned}


def exact_turns(case):
    """``amplitude * exp(i p f)`` as a function of positions: complex ``[..., R / 2]``."""
    R, factor, kind = case["R"], case["factor"], case["scaling"]
    edge = lambda n: R * math.log(TRAINED / (n * 2 * math.pi)) / (2 * math.log(10000.0))
    low, high = max(math.floor(edge(32)), 0), min(math.ceil(edge(1)), R - 1)
    f = []
    for i in range(R // 2):
        whole = math.exp(-2 * i / R * math.log(10000.0))
        if kind == "linear":
            whole /= factor
        elif kind == "yarn":
            share = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            whole = share * whole / factor + (1 - share) * whole
        f.append(whole)
    amplitude = 1 + math.log(factor) / 10 if kind == "yarn" else 1.0
    f = torch.tensor(f, dtype=torch.float64, device=DEV)
    return lambda p: torch.polar(torch.full_like(f, amplitude), p.double()[..., None] * f)


def exact_rotated(case, x, turn):
    """x ``[H, n, D]`` as complex pairs times ``turn`` ``[n, R / 2]``, in 64 bits."""
    R, x = case["R"], x.double()
    first, second = ((slice(0, R, 2), slice(1, R, 2)) if case["interleaved"]
                     else (slice(0, R // 2), slice(R // 2, R)))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x = x.clone()
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    kind, B = case["kind"], case["B"]
    if kind == "rotate":
        turns, at = exact_turns(case), torch.arange(case["N"], device=DEV)
        of = [turns(at if s["positions"] is None else s["positions"][b]) for b in range(B)]
        whole = lambda x, back: torch.stack(
            [exact_rotated(case, x[b], of[b].conj() if back else of[b]) for b in range(B)])
        out = [whole(s["q"], False), whole(s["k"], False)]
        return out + ([whole(s["gq"], True), whole(s["gk"], True)] if case["train"] else [])
    if kind == "append":
        turns, T, S, pages = exact_turns(case), case["T"], case["S"], s["pages"].double()
        out = [torch.empty(x.shape, dtype=torch.float64, device=DEV) for x in s["q"]]
        for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
            at = torch.arange(n, n + T, device=DEV)
            turn = turns(at)
            page, place = s["table"][b].long()[at[:c] // S], at[:c] % S
            for layer in range(case["L"]):
                out[layer][b] = exact_rotated(case, s["q"][layer, b], turn)
                k = exact_rotated(case, s["new"][2 * layer, b], turn)
                pages[2 * layer][page, :, place] = k[:, :c].transpose(0, 1)
                pages[2 * layer + 1][page, :, place] = s["new"][2 * layer + 1, b, :, :c].double().transpose(0, 1)
        return out + [pages]
    if kind == "attend":
        out, lse = [], []
        for b in range(B):
            n, S = int(s["lengths"][b]), case["S"]
            at = torch.arange(n, device=DEV)
            page = s["table"][b].long()[at // S]
            at, page = (at % S)[page >= 0], page[page >= 0]
            for h in range(case["Hkv"]):
                k, v = s["k"][page, h, at].double(), s["v"][page, h, at].double()
                group = case["H"] // case["Hkv"]
                z = s["q"][b, h * group:(h + 1) * group, 0].double() @ k.T * case["D"] ** -0.5
                out.append(torch.softmax(z, 1) @ v)
                lse.append(torch.logsumexp(z, 1))
        return [torch.stack(out).view(B, case["H"], 1, case["D"]), torch.stack(lse).view(B, case["H"], 1)]
    x = s["logits"].double()
    V, T = case["V"], case["T"]
    for b in range(B):
        n, given = int(s["lengths"][b]), int(s["prompts"][b])
        words = s["history"][b, :n].long()
        prompt = torch.bincount(words[:given], minlength=V) > 0
        made = torch.bincount(words[given:], minlength=V)
        r, p, f = (float(s[k][b]) for k in ("repetition", "presence", "frequency"))
        up = s["parents"][b].tolist() if T > 1 else None
        for i in range(T):
            count, j = made.clone(), i
            while up is not None and j >= 0:
                count[s["drafts"][b, j]] += 1
                j = up[j]
            row = x[b, i]
            row = torch.where(prompt | (count > 0), torch.where(row > 0, row / r, row * r), row)
            row = row - f * count - torch.where(count > 0, p, 0.0)
            if s["bias"] is not None:
                row[s["bias_tokens"][b].long()] += s["bias"][b].double()
            if s["allowed"] is not None:
                bit = torch.arange(V, device=DEV)
                row[(s["allowed"][b, i].long()[bit // 32] >> (bit % 32)) % 2 == 0] = -math.inf
            x[b, i] = row
    return x
