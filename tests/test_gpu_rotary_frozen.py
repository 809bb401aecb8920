"""Rotary where only one of its inputs needs gradients."""

import pytest
import torch

from cab_attention.cache import append_paged
from cab_attention.kernels import Rotary

pytestmark = pytest.mark.gpu


def rand(shape, seed, dt=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dt)


def test_one_output_alone_needs_gradients(cuda):
    """Frozen keys beside queries that are trained: their rotated form is frozen too, and goes into a cache."""
    rot = Rotary(64).to(cuda)
    q, k = rand((2, 4, 5, 64), 1).to(cuda).requires_grad_(), rand((2, 2, 5, 64), 2).to(cuda)
    rq, rk = rot(q, k)
    assert rq.requires_grad and not rk.requires_grad
    with torch.no_grad():
        want = rot(q, k)
    assert torch.equal(rq, want[0]) and torch.equal(rk, want[1])
    g = rand((2, 4, 5, 64), 3).to(cuda)
    (got,) = torch.autograd.grad(rq, q, g, retain_graph=True)
    leaf = q.detach().clone().requires_grad_()
    assert torch.equal(got, torch.autograd.grad(rot(leaf), leaf, g)[0])
    pools = [torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    table, n = torch.arange(2, dtype=torch.int32, device=cuda)[:, None], torch.zeros(2, dtype=torch.int32, device=cuda)
    append_paged(rk, rk, *pools, table, n)
    assert torch.equal(pools[0][:, :, :5], rk)
    qf, kt = q.detach(), k.clone().requires_grad_()
    rq, rk = rot(qf, kt)
    assert not rq.requires_grad and rk.requires_grad
    gk = rand((2, 2, 5, 64), 4).to(cuda)
    (back,) = torch.autograd.grad(rk, kt, gk)
    other = k.clone().requires_grad_()
    assert torch.equal(back, torch.autograd.grad(rot(other), other, gk)[0])
