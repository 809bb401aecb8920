"""Speculative decoding's entry points at calls their documentation allows and that lie off the
usual ones: strides of K and V apart, broadcast inputs, very many rows, nothing to do, inference
mode, the ends of the temperature's range, and the same bits whatever a workspace held."""

import numpy as np
import pytest
import torch

from oracle import spec_oracle as S
from test_gpu_tree_attn import DT, close, np64, rand, trees
from test_gpu_verify import check, make

pytestmark = pytest.mark.gpu


def attend(cuda, q, k, v, parents, n, **kw):
    from cab_attention.kernels import tree_attention
    return tree_attention(q, k, v, torch.tensor(parents).int().to(cuda),
                          torch.tensor(n, dtype=torch.int32).to(cuda), return_lse=True, **kw)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("H,T", [(4, 5), (4, 40), (4, 60)])
def test_strides_of_their_own(cuda, dt, H, T):
    """K as a cache of one sequence for the whole batch, V as a projection leaves it, queries
    the same for all heads."""
    B, Hkv, N, D = 3, 2, 500, 64
    q = rand((B, T, 1, D), dt, 1).transpose(1, 2).expand(B, H, T, D)
    k = rand((1, Hkv, N, D), dt, 2).expand(B, Hkv, N, D)
    v = rand((B, N, Hkv, 2 * D), dt, 3)[..., D:].transpose(1, 2)
    parents, n = trees(B, T, "tree", 3), [440, 0, 77]
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, n)
    q, k = q[:, :1].to(cuda).expand(B, H, T, D), k[:1].to(cuda).expand(B, Hkv, N, D)
    v = rand((B, N, Hkv, 2 * D), dt, 3).to(cuda)[..., D:].transpose(1, 2)
    close(*attend(cuda, q, k, v, parents, n), want, dt)


@pytest.mark.parametrize("dt,H,T", [("bf16", 64, 64), ("fp32", 32, 128), ("fp16", 255, 128)])
def test_very_many_rows(cuda, dt, H, T):
    """Thousands of rows a K / V head: as many row tiles, and one stretch for several units."""
    B, Hkv, N, D = 2, 1, 200 + T, 64
    q, k, v = rand((B, H, T, D), dt, 1), rand((B, Hkv, N, D), dt, 2), rand((B, Hkv, N, D), dt, 3)
    parents, n = trees(B, T, "roots", 3), [200, 65]
    want = S.tree_attention(np64(q), np64(k), np64(v), parents, n)
    close(*attend(cuda, q.to(cuda), k.to(cuda), v.to(cuda), parents, n), want, dt)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,H,Hkv,T,N", [(1, 32, 8, 5, 600), (2, 16, 2, 40, 3000), (8, 14, 2, 26, 4000),
                                         (16, 8, 2, 1, 5000), (300, 2, 1, 3, 200)])
def test_same_bits_whatever_memory_held(cuda, dt, B, H, Hkv, T, N):
    """A call again, its workspace and outputs in memory full of NaN or large numbers: the
    same bits, as no sum's order depends on anything but the sizes and lengths."""
    D = 128
    q, k, v = (rand(s, dt, i).to(cuda) for i, s in enumerate(((B, H, T, D), (B, Hkv, N, D), (B, Hkv, N, D))))
    parents = trees(B, T, "tree", 3)
    n = np.random.default_rng(5).integers(0, N - T + 1, B)
    first = attend(cuda, q, k, v, parents, n)
    for fill in (float("nan"), 1e30, -1e30):
        junk = [torch.full((1 << s,), fill, device=cuda) for s in (24, 22, 20, 16, 12, 10)]
        torch.cuda.synchronize()
        del junk  # (what the next call allocates)
        for a, b in zip(first, attend(cuda, q, k, v, parents, n)):
            assert torch.equal(a, b)


def test_nothing_to_do(cuda):
    """No sequences, no new rows, no nodes."""
    from cab_attention.cache import append_drafts, commit_drafts
    from cab_attention.kernels import tree_attention, verify_drafts
    f, i32 = (lambda *s: torch.zeros(s, device=cuda)), lambda *s: torch.zeros(s, dtype=torch.int32, device=cuda)
    out, lse = tree_attention(f(0, 4, 3, 64), f(0, 2, 20, 64), f(0, 2, 20, 64), i32(3) - 1, i32(0),
                              return_lse=True)
    assert out.shape == (0, 4, 3, 64) and lse.shape == (0, 4, 3)
    path, counts, token = verify_drafts(f(0, 3, 9), i32(0, 3), i32(3), f(0, 3), f(0, 9))
    assert path.shape == (0, 3) and counts.shape == token.shape == (0,)
    cache = torch.randn((2, 2, 9, 64), device=cuda)
    was = cache.clone()
    append_drafts(f(2, 2, 0, 64), f(2, 2, 0, 64), cache, cache.clone(), i32(2))
    append_drafts(f(0, 2, 3, 64), f(0, 2, 3, 64), f(0, 2, 9, 64), f(0, 2, 9, 64), i32(0))
    assert commit_drafts([cache], i32(2) + 4, i32(2, 0), i32(2) + 3).tolist() == [4, 4]
    assert commit_drafts([f(0, 2, 9, 64)], i32(0), i32(0, 3), i32(0)).shape == (0,)
    assert torch.equal(cache, was)


def test_inference_mode(cuda):
    """A step whose caches and inputs are inference tensors, inside inference mode."""
    from cab_attention.cache import append_drafts, commit_drafts
    from cab_attention.kernels import tree_attention, verify_drafts
    results = []
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            g = torch.Generator(device=cuda).manual_seed(1)
            f = lambda *s: torch.randn(s, generator=g, device=cuda)
            k, v, q = f(2, 2, 50, 64), f(2, 2, 50, 64), f(2, 4, 5, 64)
            n = torch.tensor([3, 40], dtype=torch.int32, device=cuda)
            up = torch.tensor([-1, 0, 0, 1, 3], dtype=torch.int32, device=cuda)
            append_drafts(f(2, 2, 5, 64), f(2, 2, 5, 64), k, v, n)
            out = tree_attention(q, k, v, up, n, out=torch.empty_like(q))
            tokens = torch.randint(0, 9, (2, 5), generator=g, device=cuda)
            path, counts, token = verify_drafts(f(2, 5, 9), tokens, up, f(2, 5).sigmoid(), f(2, 9).exp())
            results.append([out, path, counts, token, commit_drafts([k, v], n, path, counts), k, v])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("mode", ["point", "draft"])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 1e3, 1e6])
def test_ends_of_the_temperature(cuda, dt, mode, temperature):
    """From all weight on the largest logit to all weights alike."""
    x = make(4, 9, 3000, dt, "point", "tree", 17, temperature)
    if mode == "draft":
        g = torch.Generator().manual_seed(2)
        x["drafts"] = (x["logits"].float() + torch.randn(x["logits"].shape, generator=g)).to(DT[dt])
    check(x, cuda, margin=1e-6 if temperature < 1 or mode == "point" else 1e-4)
