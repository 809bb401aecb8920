"""A step over pages, captured and replayed, where workgroups share a sequence: the list of contexts, which the
device cuts anew in every replay, partials in the graph's own memory, and their join."""

import numpy as np
import pytest
import torch

from cab_attention.cache import append_paged
from cab_attention.kernels import Rotary, paged_attention
from oracle import paged_oracle as P
from test_gpu_paged_attn import ATOL, np64

pytestmark = pytest.mark.gpu


def i32(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def test_a_captured_step_over_parts(cuda):
    """Appending and attention over a table so long that workgroups share a sequence and their parts are joined,
    replayed while lengths move from none to one part to many, with eager work between."""
    B, H, HKV, D, S, COLUMNS = 3, 8, 2, 128, 16, 300
    rot = Rotary(D).to(cuda)
    g = torch.Generator().manual_seed(7)
    pages = B * COLUMNS + 1
    start = [torch.randn((pages, HKV, S, D), generator=g).bfloat16().to(cuda) for _ in range(2)]
    pools = [x.clone() for x in start]
    table = torch.randperm(pages, generator=g)[:B * COLUMNS].view(B, COLUMNS).int().to(cuda)
    lengths = i32([5, 0, 70], cuda)
    q, k, v = (torch.randn((B, h, 1, D), generator=g).bfloat16().to(cuda) for h in (H, HKV, HKV))

    def step():
        seen = lengths + 1
        turned = append_paged(k, v, *pools, table, lengths, rotary=rot, q=q)
        out, lse = paged_attention(turned, *pools, table, seen, return_lse=True)
        lengths.copy_(seen)
        return [out, lse]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for n, at in enumerate(([-1, 0, 4000], [3000, -1, -1], [100, 127, 128], [4799, 4798, 5], [-1, -1, -1], [600, 2000, 64])):
        for x, y in zip(pools, start):
            x.copy_(y)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        lengths.copy_(i32(at, cuda))
        table[1, 7 * n] = -1
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*captured, *pools, lengths)]
        for x, y in zip(pools, start):
            x.copy_(y)
        lengths.copy_(i32(at, cuda))
        want = step() + pools + [lengths]
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        host = [np64(x) for x in (append_paged(k, v, *[y.clone() for y in pools], table, i32(at, cuda), rotary=rot, q=q),
                                  *pools)]
        out, lse = P.attention(*host, table.cpu().numpy(), [x + 1 for x in at])
        np.testing.assert_allclose(np64(got[0]), out, atol=ATOL["bf16"], rtol=0)
