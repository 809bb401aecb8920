"""Rotary against the float64 oracle: layouts, parts of a head, odd sizes, strides, far positions,
gradients against the formula's and against differences, and the attention module that calls it."""

import numpy as np
import pytest
import torch

from cab_attention import CABAttention
from cab_attention.kernels import Rotary
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rand(shape, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(DT[dt])


def np64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, dt, x, amplitude=1.0):
    """Cosine and sine: polynomials and their argument, three roundings of 2^-24 at most, the
    amplitude one more, the two products and their sum three: 8 * 2^-24 of |x| + |y| <= 2 max |x|; the angle
    1.9e-9 rad. Then half a step of the type, of the value."""
    big = np.abs(np64(x)).max() * abs(amplitude) if x.numel() else 0.0
    np.testing.assert_allclose(np64(got), want, rtol=torch.finfo(DT[dt]).eps / 2 * (1 + 1e-6),
                               atol=2 * big * (8 * 2.0 ** -24 + 1.9e-9) + 2.0 ** -25)


def reference(rot, x, positions, inverse=False):
    f, a = P.rotary_frequencies(rot.rotary_dim, rot.base, rot.scaling)
    return P.rotary(np64(x), positions, f, a, rot.interleaved, inverse)


CASES = [  # B, H, H_kv, N, D, R
    (1, 1, 1, 1, 2, 2),           # one pair
    (2, 8, 2, 1, 128, 128),       # one token
    (3, 7, 1, 5, 64, 64),
    (2, 4, 4, 17, 128, 32),       # a part of the head
    (1, 3, 2, 70, 80, 16),        # rows of ten (16 bits) units
    (2, 2, 1, 33, 72, 48),        # an odd number of units
    (1, 5, 3, 9, 50, 22),         # nothing on 16-byte boundaries
    (2, 3, 1, 6, 7, 4),           # an odd head dim
    (1, 2, 2, 11, 512, 512),      # the widest
    (1, 2, 1, 4, 511, 510),       # the widest, value by value
    (1, 40, 8, 1100, 128, 128),   # four tokens a workgroup
    (5, 3, 3, 411, 64, 32),       # and one that ends past the last row
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_oracle(cuda, case, dt, interleaved):
    B, H, Hkv, N, D, R = case
    q, k = rand((B, N, H, D), dt, 1).transpose(1, 2), rand((B, Hkv, N, D), dt, 2)
    rot = Rotary(D, rotary_dim=R, interleaved=interleaved).to(cuda)
    at = np.broadcast_to(np.arange(N), (B, N))
    got = rot(q.to(cuda), k.to(cuda))
    for x, y in zip((q, k), got):
        assert y.shape == x.shape and y.dtype is x.dtype and y.is_contiguous() == x.is_contiguous()
        close(y, reference(rot, x, at), dt, x)
        assert torch.equal(y[..., R:].cpu(), x[..., R:])


@pytest.mark.parametrize("scaling", [dict(type="yarn", factor=4.0, original_length=4096),
                                     dict(type="bands", factor=8.0, original_length=8192),
                                     dict(type="ntk", factor=2.0), dict(type="linear", factor=8.0)],
                         ids=lambda s: s["type"])
@pytest.mark.parametrize("dt", list(DT))
def test_far_positions(cuda, scaling, dt):
    """Angles of positions up to the ends of 32 bits, one list for all or one a sequence."""
    far = np.array([[0, 1, -1, 130999, 1 << 20, 16777217, -123456789, (1 << 31) - 1],
                    [5, 4, 3, 2, 1, 0, -(1 << 31), 99999999]])
    rot = Rotary(128, scaling=scaling).to(cuda)
    q = rand((2, 3, 8, 128), dt, 3)
    for at in (far, far[1]):
        got = rot(q.to(cuda), positions=torch.tensor(at, dtype=torch.int32, device=cuda))
        # (the oracle's own product p f in 64 bits is off by 2^31 2^-53 = 2.4e-7 rad at most)
        want = reference(rot, q, np.broadcast_to(at, (2, 8)))
        slack = 2.4e-7 * 2 * np.abs(np64(q)).max() * rot.amplitude
        err = np.abs(np64(got) - want)
        assert (err <= np.abs(want) * torch.finfo(DT[dt]).eps / 2 * (1 + 1e-6) + slack
                + 2 * np.abs(np64(q)).max() * rot.amplitude * (8 * 2.0 ** -24 + 1.9e-9) + 2.0 ** -25).all()
    wide = torch.tensor(far[1], device=cuda)  # int64
    assert torch.equal(rot(q.to(cuda), positions=wide), got)


def test_strided_inputs(cuda):
    rot = Rotary(64, rotary_dim=32).to(cuda)
    qkv = rand((2, 50, 3, 6, 64), "bf16", 4).to(cuda)
    q, k = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
    got = rot(q, k)
    assert torch.equal(got[0], rot(q.contiguous())) and torch.equal(got[1], rot(k.contiguous()))
    odd = rand((2, 6, 50, 129), "bf16", 5).to(cuda)
    for x in (odd[..., 1:65], odd[..., ::2][..., :64], odd[:, :, :, :64].expand(2, 6, 50, 64),
              odd[:1, :, :, :64].expand(3, -1, -1, -1), odd[..., :64].flip(2), odd[:, :, ::3, 64:128]):
        assert torch.equal(rot(x), rot(x.clone(memory_format=torch.contiguous_format)))


def test_empty_tensors(cuda):
    rot = Rotary(64).to(cuda)
    for shape in ((0, 2, 5, 64), (2, 2, 0, 64), (2, 0, 5, 64)):
        assert rot(torch.empty(shape, device=cuda)).shape == shape
    x = rand((2, 3, 5, 64), "fp32", 1).to(cuda)
    got = rot(x, x[:, :0])
    assert torch.equal(got[0], rot(x)) and got[1].shape == (2, 0, 5, 64)


def test_infinities_stay_in_their_pair(cuda):
    rot = Rotary(64).to(cuda)
    x = rand((1, 2, 6, 64), "fp32", 1).to(cuda)
    x[0, 1, 3, 5], x[0, 0, 2, 40] = float("inf"), float("nan")
    got, clean = rot(x), rot(torch.nan_to_num(x, 0.0, 0.0))
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[0, 1, 3, [5, 37]] = True
    want[0, 0, 2, [40, 8]] = True
    assert torch.equal(bad, want) and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", list(DT))
def test_gradients(cuda, dt, interleaved):
    """Against the transpose of the rotation, with the amplitude, and a gradient whose strides are 0."""
    rot = Rotary(64, rotary_dim=48, interleaved=interleaved,
                 scaling=dict(type="yarn", factor=4.0, original_length=64)).to(cuda)
    at = np.random.default_rng(0).integers(-1000, 100000, (2, 37))
    positions = torch.tensor(at, dtype=torch.int32, device=cuda)
    q = rand((2, 37, 6, 64), dt, 1).to(cuda).transpose(1, 2).requires_grad_()
    k = rand((2, 2, 37, 64), dt, 2).to(cuda).requires_grad_()
    gq, gk = rand((2, 6, 37, 64), dt, 3), rand((2, 2, 37, 64), dt, 4)
    out = rot(q, k, positions)
    got = torch.autograd.grad(out, (q, k), (gq.to(cuda), gk.to(cuda)))
    for x, g, y in zip((q, k), (gq, gk), got):
        assert y.shape == x.shape and y.dtype is x.dtype
        close(y, reference(rot, g, at, inverse=True), dt, g, rot.amplitude)
    ones = torch.autograd.grad(rot(q, k, positions)[1].sum(), (q, k), allow_unused=True)
    assert ones[0] is None
    close(ones[1], reference(rot, torch.ones_like(gk), at, inverse=True), dt, torch.ones_like(gk), rot.amplitude)


def test_gradients_of_broadcast_inputs(cuda):
    """A key head shared by expansion: its gradient is the sum over the copies."""
    rot = Rotary(64).to(cuda)
    k = rand((2, 1, 9, 64), "fp32", 1).to(cuda).requires_grad_()
    g = rand((2, 4, 9, 64), "fp32", 2).to(cuda)
    (got,) = torch.autograd.grad(rot(k.expand(-1, 4, -1, -1)), k, g)
    # four terms of up to 5, each off by 16 * 2^-24 of it, and their sum's roundings
    np.testing.assert_allclose(np64(got), reference(rot, g, np.broadcast_to(np.arange(9), (2, 9)), True).sum(
        1, keepdims=True), atol=4 * 5 * 24 * 2.0 ** -24, rtol=0)


def test_gradient_against_differences(cuda):
    """The operator is linear: f(x + d) - f(x) = J d exactly; <g, J d> = <J^T g, d>."""
    rot = Rotary(32, rotary_dim=16).to(cuda)
    x = rand((1, 2, 5, 32), "fp32", 1).to(cuda).requires_grad_()
    d, g = rand((1, 2, 5, 32), "fp32", 2).to(cuda), rand((1, 2, 5, 32), "fp32", 3).to(cuda)
    (back,) = torch.autograd.grad(rot(x), x, g)
    with torch.no_grad():
        moved = (rot(x + d).double() - rot(x).double() - 0.0)
    # 320 terms, each with factors up to 5 that are off by some 16 * 2^-24 * 10
    assert abs(float((g.double() * moved).sum() - (back.double() * d.double()).sum())) < 320 * 5 * 160 * 2.0 ** -24


def test_second_order_and_changed_positions(cuda):
    rot = Rotary(64).to(cuda)
    x = rand((1, 2, 5, 64), "fp32", 1).to(cuda).requires_grad_()
    g = rand((1, 2, 5, 64), "fp32", 2).to(cuda).requires_grad_()
    (first,) = torch.autograd.grad(rot(x), x, g, create_graph=True)
    (second,) = torch.autograd.grad(first, g, x.detach())  # d<R^T g, x> / dg = R x
    assert torch.equal(second, rot(x.detach()))
    at = torch.arange(5, dtype=torch.int32, device=cuda)
    y = rot(x, positions=at)
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals_on_the_device(cuda):
    rot = Rotary(64).to(cuda)
    x = rand((2, 2, 5, 64), "bf16", 1).to(cuda)
    with pytest.raises(ValueError, match="positions"):
        rot(x, positions=torch.arange(4, device=cuda))
    with pytest.raises(TypeError, match="positions"):
        rot(x, positions=torch.arange(5.0, device=cuda))
    with pytest.raises(TypeError):
        rot(x.double())
    with pytest.raises(RuntimeError):
        Rotary(64)(x)  # its turns are on the host
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.vmap(lambda y: rot(y[None]))(x)


def test_captured_forward_and_backward(cuda):
    """Replays follow inputs and positions, with an eager graph of other leaves alive."""
    rot = Rotary(128).to(cuda)
    q = rand((2, 4, 33, 128), "bf16", 1).to(cuda).requires_grad_()
    g = rand((2, 4, 33, 128), "bf16", 2).to(cuda)
    at = torch.arange(33, dtype=torch.int32, device=cuda)
    eager = rand((2, 4, 33, 128), "bf16", 3).to(cuda).requires_grad_()
    alive = rot(eager, positions=at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rot(q, positions=at)
        (back,) = torch.autograd.grad(y, q, g)
    for n in range(4):
        with torch.no_grad():
            q.copy_(rand((2, 4, 33, 128), "bf16", 10 + n))
            g.copy_(rand((2, 4, 33, 128), "bf16", 20 + n))
        at.copy_(torch.arange(33) * (n + 1))
        graph.replay()
        torch.cuda.synchronize()
        free = q.detach().clone().requires_grad_()
        want = rot(free, positions=at.clone())
        assert torch.equal(y, want) and torch.equal(back, torch.autograd.grad(want, free, g)[0])
    del alive


def test_on_another_stream(cuda):
    rot = Rotary(64).to(cuda)
    side = torch.cuda.Stream()
    x = rand((1, 4, 3000, 64), "fp16", 1).to(cuda)
    want = rot(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = x + 0.0
        got = rot(z)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_attention_module(cuda, dt):
    """CABAttention(rotary=..) is attention of the rotated queries and keys; without it nothing changes."""
    torch.manual_seed(0)
    rot = Rotary(64, rotary_dim=32)
    module = CABAttention(256, 4, sparsity=0.5, causal=True, rotary=rot).to(cuda, DT[dt])
    plain = CABAttention(256, 4, sparsity=0.5, causal=True).to(cuda, DT[dt])
    plain.load_state_dict(module.state_dict())
    x = rand((2, 300, 256), dt, 5).to(cuda)
    at = torch.arange(7, 307, device=cuda)
    with torch.no_grad():
        y = module(x, positions=at)
        q, k, v = module.qkv(x).view(2, 300, 3, 4, 64).permute(2, 0, 3, 1, 4)
        want = plain.proj(plain.attend(rot(q, positions=at), rot(k, positions=at), v).transpose(1, 2).reshape(2, 300, 256))
        assert torch.equal(y, want)
        assert not torch.equal(module(x), plain(x))
        zero = torch.zeros(300, dtype=torch.int32, device=cuda)
        assert torch.equal(module(x, positions=zero), plain(x))


def test_backward_after_the_module_moved(cuda):
    """What the forward pass took is kept for the backward pass, whatever becomes of the module."""
    rot = Rotary(64).to(cuda)
    x = rand((1, 2, 5, 64), "fp32", 1).to(cuda).requires_grad_()
    g = rand((1, 2, 5, 64), "fp32", 2).to(cuda)
    (want,) = torch.autograd.grad(rot(x), x, g)
    y = rot(x)
    rot.cpu()
    rot.amplitude = 3.0
    (got,) = torch.autograd.grad(y, x, g)
    assert torch.equal(got, want)
    rot.turns = rot.turns.float().to(cuda)
    with pytest.raises(RuntimeError, match="turns"):
        rot(x)
