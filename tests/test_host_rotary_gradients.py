"""Which of Rotary's outputs need gradients, without a GPU (the kernel call replaced)."""

import pytest
import torch

from cab_attention.kernels import Rotary, rotary


@pytest.mark.parametrize("which", [(True, False), (False, True), (True, True)])
def test_outputs_need_the_gradients_that_their_inputs_need(monkeypatch, which):
    calls = []

    def turn(plan, turns, positions, inverse, tensors):
        calls.append((inverse, len(tensors)))
        return [x * (-2.0 if inverse else 2.0) for x in tensors]

    monkeypatch.setattr(rotary, "_turn", turn)
    monkeypatch.setattr(rotary, "_plain", lambda *a: None)
    rot = Rotary(128, rotary_dim=64)
    q, k = (torch.ones((1, 2, 3, 128), requires_grad=need) for need in which)
    out = rot(q, k)
    assert tuple(y.requires_grad for y in out) == which and calls == [(False, 2)]
    for x, y in zip((q, k), out):
        if x.requires_grad:
            (g,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
            assert torch.equal(g, torch.full_like(x, -2.0))
    assert all(c == (True, 1) for c in calls[1:])
