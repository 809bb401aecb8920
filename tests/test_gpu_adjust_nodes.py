"""adjust_logits where a workgroup serves several rows of a sequence: counts taken off again between a
tree's nodes, rows at alignments of their own, groups that are not full, in place."""

import pytest
import torch

from cab_attention.kernels import adjust_logits
from test_gpu_adjust import DT, adjust_like, call, check, setup

pytestmark = pytest.mark.gpu

# A workgroup takes ceil(T / g) rows with g = ceil(ceil(768 / B) / stretches of 8192 tokens).
CASES = [  # B, T, V; rows a workgroup, of the last one
    (64, 47, 1000),    # 4, 3
    (63, 30, 1215),    # 3, 3; odd rows
    (200, 10, 333),    # 3, 1
    (768, 5, 100),     # all
    (40, 16, 20001),   # 3, 1; three stretches
    (24, 256, 301),    # 8; the most nodes
]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("biases, masked", [(0, False), (5, True)])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_several_rows_a_workgroup(cuda, case, biases, masked, tree, dt):
    B, T, V = case
    a = setup(B, T, V, 40, dt, seed=V, biases=biases, masked=masked, tree=tree)
    got = call(a, cuda)
    check(a, got, dt)
    x = a["logits"].to(cuda)
    own = dict(a, logits=x)
    assert call(own, cuda, out=x) is x and torch.equal(x, got)


@pytest.mark.parametrize("dt", list(DT))
def test_rows_at_any_alignment(cuda, dt):
    """Odd rows of a larger tensor, so that each row's 16-byte units begin elsewhere: to a new tensor, to one laid
    out otherwise, in place."""
    B, T, V = 64, 47, 1001
    a = setup(B, T, V, 60, dt, seed=1, biases=5, masked=True, tree=True)
    want = call(a, cuda)
    check(a, want, dt)
    for lead in (0, 1, 5):
        room = torch.zeros((B, T + 1, V + 12), dtype=DT[dt], device=cuda)
        view = room[:, 1:, lead:lead + V]
        view.copy_(a["logits"])
        assert torch.equal(adjust_like(a, cuda, view), want)
        out = torch.full((B, T, V + 6), 9.0, dtype=DT[dt], device=cuda)
        to = out[..., 3:V + 3]
        adjust_like(a, cuda, view, out=to)
        assert torch.equal(to, want)
        to.fill_(9.0)
        assert (out == 9.0).all()
        adjust_like(a, cuda, view, out=view)
        assert torch.equal(view, want)
        view.zero_()
        assert not room.any()


@pytest.mark.parametrize("T", [47, 48])
def test_a_token_of_one_node_alone(cuda, T):
    """Every node a child of the first, with a token of its own: it counts for its node and no other; in a
    chain it counts for all behind it."""
    B, V = 64, 1000
    x = torch.zeros((B, T, V), device=cuda)
    drafts = (torch.arange(T, device=cuda) * 7 + torch.arange(B, device=cuda)[:, None]) % V
    at = torch.arange(T, device=cuda)
    star, chain = torch.zeros(T, dtype=torch.int32, device=cuda), (at - 1).int()
    star[0] = -1
    for parents in (star, chain):
        got = adjust_logits(x, frequency=0.5, presence=0.25, drafts=drafts, parents=parents)
        line = torch.eye(T, dtype=torch.bool, device=cuda)
        line = line | (at == 0) if parents is star else torch.tril(torch.ones_like(line))
        want = torch.zeros_like(x)
        want.scatter_(2, drafts[:, None].expand(B, T, T), -0.75 * line[None].expand(B, T, T).float())
        assert torch.equal(got, want)
    same = adjust_logits(x, frequency=0.5, drafts=torch.full_like(drafts, 9), parents=chain)
    assert torch.equal(same[:, :, 9], (-0.5 * (at + 1)).expand(B, T)) and int((same != 0).sum()) == B * T
