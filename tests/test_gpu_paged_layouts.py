"""Rotary, append_paged and paged_attention on layouts at the edge of "any strides": windows that slide over one
row, rows of one value, dims of one place with strides of no meaning."""

import pytest
import torch

from cab_attention.cache import append_paged
from cab_attention.kernels import Rotary, paged_attention

pytestmark = pytest.mark.gpu


def rand(shape, seed, dt=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dt)


def test_windows_that_slide_over_a_row(cuda):
    """Rows at a stride of one value, fewer than a head's values: an output cannot be laid out like them."""
    rot = Rotary(64).to(cuda)
    x = rand(70, 1).to(cuda).unfold(0, 64, 1)[None, None]  # [1, 1, 7, 64]
    flat = x.contiguous()
    assert torch.equal(rot(x), rot(flat))
    both = rot(x, x)
    assert torch.equal(both[0], rot(flat)) and torch.equal(both[1], rot(flat))
    leaf = flat.clone().requires_grad_()
    (got,) = torch.autograd.grad(rot(leaf), leaf, x)
    (want,) = torch.autograd.grad(rot(leaf), leaf, flat)
    assert torch.equal(got, want)
    pools = [torch.zeros((2, 1, 16, 64), dtype=torch.bfloat16, device=cuda) for _ in range(4)]
    table, n = torch.tensor([[1]], dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    a = append_paged(x, x, *pools[:2], table, n, rotary=rot, q=x)
    b = append_paged(flat, flat, *pools[2:], table, n, rotary=rot, q=flat)
    assert torch.equal(a, b) and torch.equal(a, rot(flat))
    assert all(torch.equal(y, z) for y, z in zip(pools[:2], pools[2:])) and pools[0].any()


def test_rows_of_one_value(cuda):
    """D = 1: the last stride has no meaning."""
    wide = rand((2, 3, 5, 7), 1).to(cuda)
    k, v = wide[..., ::7], wide[..., 3::7]
    assert k.shape == v.shape == (2, 3, 5, 1) and k.stride(3) == 7
    room = torch.zeros((6, 3, 4, 5), dtype=torch.bfloat16, device=cuda)
    pools, others = [room[..., 1::5], room[..., 3::5]], [torch.zeros((6, 3, 4, 1), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    table = torch.tensor([[4, 0], [2, 5]], dtype=torch.int32, device=cuda)
    n = torch.tensor([1, 3], dtype=torch.int32, device=cuda)
    append_paged(k, v, *pools, table, n)
    append_paged(k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format),
                 *others, table, n)
    for x, y in zip(pools, others):
        assert torch.equal(x, y) and x.any()
    assert not room[..., [0, 2, 4]].any()


def test_dims_of_one_place(cuda):
    """One head, one page, one place a page, at strides off every boundary."""
    q = rand((1, 2, 1, 64), 1).to(cuda)
    k, v = (rand(64 * 40, s).to(cuda) for s in (2, 3))
    odd = lambda x: x.as_strided((3, 1, 1, 64), (64, 3, 1 << 27, 1))
    even = lambda x: x[:192].view(3, 1, 1, 64)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=cuda)
    n = torch.tensor([3], dtype=torch.int32, device=cuda)
    want = paged_attention(q, even(k), even(v), table, n)
    assert torch.equal(paged_attention(q, odd(k), odd(v), table, n), want)
    one = lambda x: x[:1024].as_strided((1, 1, 16, 64), (5, 3, 64, 1))
    flat = lambda x: x[:1024].view(1, 1, 16, 64)
    want = paged_attention(q, flat(k), flat(v), table[:, 1:2], n)
    assert torch.equal(paged_attention(q, one(k), one(v), table[:, 1:2], n), want)
