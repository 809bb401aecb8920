"""Rotary as a module, without a GPU: frequencies after a start on the meta device or in empty memory."""

import copy

import pytest
import torch

from cab_attention import CABAttention
from cab_attention.kernels import Rotary


def dirty():
    """Memory that a later allocation of a module's buffers may be given."""
    for _ in range(50):
        torch.full((64,), 7, dtype=torch.int64)


def make():
    return Rotary(128, rotary_dim=64, base=5e5, scaling=dict(type="bands", factor=8.0, original_length=8192))


def test_frequencies_after_a_start_on_the_meta_device():
    want = make().turns
    with torch.device("meta"):
        late = make()
        module = CABAttention(512, 4, rotary=make())
    assert late.turns.is_meta and late.frequencies == make().frequencies
    dirty()
    assert torch.equal(late.to_empty(device="cpu").turns, want)
    plain = CABAttention(512, 4, rotary=make())
    dirty()
    module.to_empty(device="cpu").load_state_dict(plain.state_dict())
    assert torch.equal(module.rotary.turns, want) and module.rotary.plan()[1] is module.rotary.turns


def test_frequencies_in_empty_memory():
    want, rot = make().turns, make()
    dirty()
    assert torch.equal(rot.to_empty(device="cpu").turns, want)
    rot.turns.zero_()
    rot.reset_parameters()
    assert torch.equal(rot.turns, want)


def test_a_module_that_stays_keeps_its_buffer():
    rot = make()
    at = rot.turns
    rot.to("cpu").half().float().eval()
    assert rot.turns is at and at._version == rot.turns._version
    assert torch.equal(copy.deepcopy(rot).turns, at)
    rot.type(torch.float32)  # converts every buffer: refused where it is used
    with pytest.raises(RuntimeError, match="turns"):
        rot.plan()
