"""verify_drafts against the float64 oracle: paths, counts and next tokens equal, over
trees, modes, types and vocabularies, with masked, infinite and NaN logits. Every
decision of these inputs is further from its border than the kernel's error (see
MARGIN), which the tests check of the oracle's values first."""

import numpy as np
import pytest
import torch

from oracle import spec_oracle as S

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# The kernel's weights are within 4 fp32 roundings of exp (2.4e-7), sums of up to 8 of
# them in fp32 add 3 more; differences p - a q within a factor 100 of p keep 1e-4.
MARGIN = 1e-6


def tree(T, shape, rng):
    if shape == "chain":
        return [-1] + list(range(T - 1))
    if shape == "star":
        return [-1] + [0] * (T - 1)
    return [-1] + [int(i * rng.random()) for i in range(1, T)]


def make(B, T, V, dt, mode, shape, seed, temperature):
    rng = np.random.default_rng(seed)
    parents = np.array([tree(T, shape, rng) for _ in range(B)])
    logits = rng.standard_normal((B, T, V)).astype(np.float32)
    top = rng.integers(0, V, (B, T, 4))
    np.put_along_axis(logits, top, (5 + 3 * rng.random((B, T, 4))).astype(np.float32), 2)
    drafts = logits + 0.7 * rng.standard_normal((B, T, V)).astype(np.float32)
    tokens = np.zeros((B, T), np.int64)
    for b in range(B):
        for i in range(1, T):
            p = parents[b, i]
            if mode == "draft":
                e = np.exp((drafts[b, p] - drafts[b, p].max()) / temperature)
                tokens[b, i] = rng.choice(V, p=e / e.sum())
            else:
                tokens[b, i] = top[b, p, rng.integers(0, 4)]
    to = lambda x: torch.from_numpy(x).to(DT[dt])
    return dict(logits=to(logits), drafts=to(drafts) if mode == "draft" else None,
                tokens=torch.from_numpy(tokens), parents=torch.from_numpy(parents).int(),
                uniforms=torch.from_numpy(rng.random((B, T)).astype(np.float32)),
                noise=torch.from_numpy(rng.exponential(size=(B, V)).astype(np.float32)),
                temperature=temperature)


def check(x, cuda, margin=MARGIN):
    from cab_attention.kernels import verify_drafts
    B, T, V = x["logits"].shape
    want = []
    for b in range(B):
        up = x["parents"] if x["parents"].dim() == 1 else x["parents"][b]
        path, token, m = S.verify(x["logits"][b].float().numpy(), x["tokens"][b].tolist(), up.tolist(),
                                  x["uniforms"][b].numpy(), x["noise"][b].numpy(), x["temperature"],
                                  None if x["drafts"] is None else x["drafts"][b].float().numpy())
        assert m > margin, f"sequence {b}: a decision lies {m} from its border"
        want.append((path, token))
    dev = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    path, counts, token = verify_drafts(dev["logits"], dev["tokens"], dev["parents"], dev["uniforms"],
                                        dev["noise"], temperature=x["temperature"],
                                        draft_logits=dev["drafts"])
    assert path.dtype == torch.int32 and counts.dtype == torch.int32 and token.dtype == torch.int64
    for b, (p, t) in enumerate(want):
        assert path[b].tolist() == p + [-1] * (T - len(p)), b
        assert int(counts[b]) == len(p) and int(token[b]) == t, b
    return [len(p) for p, _ in want]


@pytest.mark.parametrize("T,V,shape", [(1, 1, "tree"), (1, 1000, "tree"), (2, 7, "chain"),
                                       (5, 32000, "chain"), (9, 8193, "star"), (26, 50001, "tree"),
                                       (64, 4096, "tree"), (65, 1023, "star"), (256, 333, "tree"),
                                       (256, 64, "chain")])
@pytest.mark.parametrize("mode", ["greedy", "point", "draft"])
@pytest.mark.parametrize("dt", list(DT))
def test_against_oracle(cuda, T, V, shape, mode, dt):
    B = 2 if V > 40000 else 5
    x = make(B, T, V, dt, mode, shape, T * 7 + V, {"greedy": 0.0, "point": 0.7, "draft": 1.2}[mode])
    check(x, cuda)


@pytest.mark.parametrize("mode", ["greedy", "point", "draft"])
def test_rows_one_after_another(cuda, mode):
    """Logits past the size up to which all rows' statistics are taken."""
    from cab_attention.kernels import verify_drafts
    g = torch.Generator(device=cuda).manual_seed(8)
    B, T, V = 4, 32, 600_001
    t = 0.0 if mode == "greedy" else 0.8
    logits = torch.randn((B, T, V), generator=g, device=cuda)  # 307 MB
    top = torch.randint(0, V, (B, T, 3), generator=g, device=cuda)
    logits.scatter_(2, top, 14 + 3 * torch.rand((B, T, 3), generator=g, device=cuda))
    logits[:, :, -7:] = -torch.inf
    drafts = None
    if mode == "draft":
        drafts = logits + 0.3 * torch.randn((B, T, V), generator=g, device=cuda)
    parents = torch.tensor([-1] + [i // 2 for i in range(T - 1)], dtype=torch.int32)
    tokens = top[:, [max(p, 0) for p in parents.tolist()], 0].clone()
    tokens[:, 1::2] = torch.randint(0, V, (B, T // 2), generator=g, device=cuda)
    if mode == "greedy":
        tokens[:, 2::2] = logits.argmax(2)[:, parents[2::2].tolist()]
    u = torch.rand((B, T), generator=g, device=cuda)
    noise = torch.empty((B, V), device=cuda).exponential_(generator=g)
    got = verify_drafts(logits, tokens, parents.to(cuda), u, noise, t, drafts)
    for b in range(B):
        path, token, m = S.verify(logits[b].cpu().numpy(), tokens[b].tolist(), parents.tolist(),
                                  u[b].cpu().numpy(), noise[b].cpu().numpy(), t,
                                  None if drafts is None else drafts[b].cpu().numpy())
        assert m > MARGIN
        assert got[0][b, :len(path)].tolist() == path and int(got[1][b]) == len(path)
        assert int(got[2][b]) == token


@pytest.mark.parametrize("mode", ["greedy", "point"])
def test_equal_scores_go_to_the_lowest_index(cuda, mode):
    """Equal logits (and equal noise) far apart in a long row, in every slice of it."""
    from cab_attention.kernels import verify_drafts
    V = 130_000
    logits = torch.zeros((1, 1, V), device=cuda)
    logits[0, 0, [V - 1, 77_777, 31_000, 65_536]] = 3.0
    ones = torch.ones((1, V), device=cuda)
    token = verify_drafts(logits, torch.zeros((1, 1), dtype=torch.int64, device=cuda),
                          torch.tensor([-1], device=cuda), torch.zeros((1, 1), device=cuda), ones,
                          0.0 if mode == "greedy" else 0.7)[2]
    assert token.tolist() == [31_000]


@pytest.mark.parametrize("mode", ["greedy", "point", "draft"])
def test_long_walks(cuda, mode):
    """Certain drafts: the whole chain is taken."""
    x = make(3, 40, 500, "fp32", mode, "chain", 5, 0.0 if mode == "greedy" else 1.0)
    for i in range(1, 40):
        x["logits"][:, i - 1].scatter_(1, x["tokens"][:, i:i + 1], 60.0)
    if x["drafts"] is not None:
        x["drafts"] = x["logits"].clone()
        x["uniforms"].clamp_(max=0.999)
    assert check(x, cuda) == [40] * 3


@pytest.mark.parametrize("mode", ["greedy", "point", "draft"])
@pytest.mark.parametrize("dt", list(DT))
def test_masked_rows(cuda, mode, dt):
    """-inf, the type's lowest value, NaN and +inf logits; rows of nothing else."""
    t = 0.0 if mode == "greedy" else 0.9
    x = make(8, 6, 700, dt, mode, "star", 11, t)
    low = torch.finfo(DT[dt]).min
    lo = x["logits"]
    lo[0, :, 300:] = -torch.inf
    lo[1, :, 1::2] = low
    lo[2, :, 5:9] = torch.nan
    lo[3] = -torch.inf           # no weight at all: next token -1
    lo[4] = torch.nan
    lo[5] = low                  # all alike
    lo[6, :, 17] = torch.inf     # all the weight on one
    lo[6, :, 400] = torch.inf    # ... two
    lo[7, :, :] = -torch.inf     # a single token left, and it is the draft
    lo[7, 0, 55] = 1.0
    x["tokens"][7, 3] = 55
    x["tokens"][2, 2] = 6
    if x["drafts"] is not None:
        x["drafts"][2, :, 5:9] = torch.nan
        x["drafts"][1, :, 1::2] = low
        x["drafts"][0, 0] = -torch.inf
    from cab_attention.kernels import verify_drafts
    check(x, cuda)
    dev = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    _, counts, token = verify_drafts(dev["logits"], dev["tokens"], dev["parents"], dev["uniforms"],
                                     dev["noise"], temperature=t, draft_logits=dev["drafts"])
    assert token[3] == -1 and token[4] == -1 and counts[3] == 1 and counts[4] == 1


@pytest.mark.parametrize("mode", ["point", "draft"])
def test_nothing_left(cuda, mode):
    """All weight on rejected drafts (uniforms past 1 reject everything): the next token
    comes from the target's own row."""
    x = make(4, 4, 50, "fp32", mode, "star", 3, 1.0)
    x["logits"][:] = -torch.inf
    x["logits"][:, :, 10:13] = torch.tensor([1.0, 2.0, 0.5])
    x["tokens"][:, 1:] = torch.tensor([10, 11, 12])
    if x["drafts"] is not None:
        x["drafts"] = x["logits"].clone()
    x["uniforms"][:] = 2.0
    assert check(x, cuda) == [1] * 4


def test_bad_drafts_are_passed_over(cuda):
    """Tokens outside the vocabulary, absent nodes, parents that are none, the same token
    twice among siblings, NaN numbers, noise that is no sample."""
    for mode in ("greedy", "point", "draft"):
        x = make(4, 12, 300, "bf16", mode, "tree", 21, 0.0 if mode == "greedy" else 0.8)
        x["tokens"][:, 1] = torch.tensor([-1, 300, 1 << 40, -(1 << 50)])
        x["parents"][0, 5:] = -2
        x["parents"][1, 4] = 4
        x["parents"][1, 6] = 11
        x["parents"][2, 3:7] = 0
        x["tokens"][2, 3:7] = x["tokens"][2, 3]
        x["uniforms"][3, 2] = torch.nan
        x["noise"][3, ::3] = torch.nan
        x["noise"][2, ::3] = -1.0
        x["noise"][1, 7] = 0.0 if mode == "point" else 1.0
        check(x, cuda)


@pytest.mark.parametrize("mode", ["greedy", "point", "draft"])
def test_layouts(cuda, mode):
    """One tree for all, logits as a slice of longer rows (odd alignment) and of more
    nodes, int32 tokens, strided parents."""
    x = make(3, 10, 501, "bf16", mode, "tree", 31, 0.0 if mode == "greedy" else 1.0)
    x["parents"] = x["parents"][0].contiguous()
    base = torch.randn((3, 13, 600)).bfloat16()
    base[:, 2:12, 3:504] = x["logits"]
    x["logits"] = base[:, 2:12, 3:504]
    x["tokens"] = x["tokens"].int()
    check(x, cuda)
    x["logits"] = x["logits"].transpose(1, 2).contiguous().transpose(1, 2)  # last dim apart
    x["parents"] = torch.stack([x["parents"]] * 2, 1)[:, 0]
    check(x, cuda)


def test_samples_the_target(cuda):
    """The next token's frequencies, over many draws, are the target's whatever the drafts'
    distribution: chi-square of 8 tokens within 5 sigma (7 degrees of freedom: mean 7,
    variance 14), of drafts accepted and of tokens drawn after rejections together."""
    from cab_attention.kernels import verify_drafts
    g = torch.Generator(device=cuda).manual_seed(4)
    n, V, T = 100_000, 8, 4
    p = torch.tensor([2.0, 1.0, 0.0, 0.5, -1.0, 1.5, -0.5, 0.2], device=cuda)
    q = torch.tensor([0.0, 2.0, 1.0, -1.0, 0.5, 0.3, 1.2, -2.0], device=cuda)
    logits = p.expand(n, T, V).contiguous()
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=cuda)
    u = torch.rand((n, T), generator=g, device=cuda)
    noise = torch.empty((n, V), device=cuda).exponential_(generator=g)
    for drafts in (None, q.expand(n, T, V).contiguous()):
        if drafts is None:
            tokens = torch.tensor([0, 1, 5, 2], device=cuda).expand(n, T).contiguous()
        else:
            e = torch.empty((n, T, V), device=cuda).exponential_(generator=g)
            tokens = (torch.softmax(q, 0) / e).argmax(2)
        path, counts, token = verify_drafts(logits, tokens, parents, u, noise, draft_logits=drafts)
        first = torch.where(counts > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token)
        seen = torch.bincount(first, minlength=V).double()
        want = torch.softmax(p.double(), 0) * n
        chi = float(((seen - want) ** 2 / want).sum())
        assert chi < 7 + 5 * 14 ** 0.5, (chi, seen.tolist(), want.tolist())
