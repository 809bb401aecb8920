"""Rotary positions (``cab_rotary``): queries and keys turned by their positions, with
gradients. The reference takes queries and keys as they come and has no counterpart."""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import torch

from .. import _native as nat

# 2^150 / (2 pi), from 2 pi to 53 digits: turns are formed to the last of 64 bits.
_TURN = (10 ** 53 << 150) // 628318530717958647692528676655900576839433879875021164


def _turns(x: float) -> int:
    """``x / (2 pi)`` modulo 1 in units of 2^-64, as the int64 of the same bits."""
    n, d = x.as_integer_ratio()  # (d: a power of two)
    t = (n * _TURN >> d.bit_length() + 84) + 1 >> 1 & (1 << 64) - 1
    return t - (1 << 64) if t >> 63 else t


def _frequencies(dim: int, base: float, scaling: Optional[dict]):
    """Radians a position for each of ``dim / 2`` pairs (Python floats), and the amplitude."""
    scaling = dict(scaling or {"type": "none"})
    kind = scaling.pop("type", None)
    known = {"none": (), "linear": ("factor",), "ntk": ("factor",),
             "yarn": ("factor", "original_length", "beta_fast", "beta_slow", "amplitude"),
             "bands": ("factor", "original_length", "low", "high")}
    if kind not in known or not set(scaling) <= set(known[kind]):
        raise ValueError(f"scaling must be one of {list(known)} with its values; got type {kind!r} "
                         f"and {sorted(scaling)}")
    needs = set(known[kind][:2]) - set(scaling)
    if needs:
        raise ValueError(f"scaling of type {kind!r} needs {sorted(needs)}")
    for name, x in scaling.items():
        if not math.isfinite(x) or (x <= 0 and name != "amplitude"):
            raise ValueError(f"scaling: {name} must be finite and positive; got {x}")
    factor = float(scaling.get("factor", 1.0))
    if kind == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    amplitude = 1.0
    if kind == "linear":
        f = [x / factor for x in f]
    elif kind == "yarn":
        length = float(scaling["original_length"])
        pair = lambda turns: dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(pair(scaling.get("beta_fast", 32.0))), 0)
        high = min(math.ceil(pair(scaling.get("beta_slow", 1.0))), dim - 1)
        for i, x in enumerate(f):
            ramp = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            f[i] = x / factor * ramp + x * (1.0 - ramp)
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
        amplitude = float(scaling.get("amplitude", amplitude))
    elif kind == "bands":
        length = float(scaling["original_length"])
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        if low >= high:
            raise ValueError(f"scaling: low must be below high; got {low} and {high}")
        for i, x in enumerate(f):
            turns = length * x / (2 * math.pi)
            kept = min(1.0, max(0.0, (turns - low) / (high - low)))
            f[i] = (1.0 - kept) * x / factor + kept * x
    return f, amplitude


@functools.lru_cache(maxsize=1024)
def _joined(*strides: tuple):
    return nat.stride_array(sum(strides, ()))


def _plain(fn: str, *tensors: torch.Tensor) -> None:
    """:func:`nat.plain_index` for tensors whose gradients may be recorded."""
    nat.require_device(*tensors)
    if not nat.addressable(*tensors):
        raise RuntimeError(f"{fn} takes plain tensors outside transforms, tracing and modes")


def _turn(plan: tuple, turns: torch.Tensor, positions, inverse: bool, tensors):
    """plan: (rotary_dim, interleaved, amplitude)."""
    tensors = [x if x.stride(3) == 1 else x.contiguous() for x in tensors]
    outs = [nat.empty_rows_like(x) for x in tensors]
    n = len(tensors)
    B, _, N, D = tensors[0].shape
    array = ctypes.c_void_p * n
    dev = tensors[0].get_device()
    with nat.at_index(dev):
        st = nat.load().cab_rotary(
            n, array(*[x.data_ptr() for x in tensors]), array(*[x.data_ptr() for x in outs]),
            nat.dtype_code(tensors[0]), B, nat.stride_array(tuple(x.shape[1] for x in tensors)), N, D,
            _joined(*[x.stride() for x in tensors]), _joined(*[x.stride() for x in outs]),
            nat.ptr(positions), 0 if positions is None or positions.dim() == 1 else N,
            turns.data_ptr(), *plan, inverse, nat.raw_stream(dev))
    if st:
        nat.check("cab_rotary", st)
    return outs


class _Turned(torch.autograd.Function):
    """One or two tensors turned together. A rotation's gradient is the rotation back."""

    @staticmethod
    def forward(ctx, plan, turns, positions, inverse, *tensors):
        ctx.plan, ctx.inverse = plan, inverse
        ctx.set_materialize_grads(False)
        # (changed in place before the backward pass: an error, not other angles)
        ctx.save_for_backward(turns, positions)
        outs = tuple(_turn(plan, turns, positions, inverse, [x.detach() for x in tensors]))
        # (a frozen key's turned form is frozen too)
        ctx.mark_non_differentiable(*[y for y, need in zip(outs, ctx.needs_input_grad[4:]) if not need])
        return outs

    @staticmethod
    def backward(ctx, *grads):
        turns, positions = ctx.saved_tensors
        at = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[4 + i]]
        out = [None] * len(grads)
        if at:
            given = [grads[i] for i in at]
            _plain("Rotary's gradient", *given)
            back = (ctx.plan, turns, positions, not ctx.inverse)
            # (recorded only for gradients of gradients)
            turned = _Turned.apply(*back, *given) if torch.is_grad_enabled() else _turn(*back, given)
            for i, x in zip(at, turned):
                out[i] = x
        return (None, None, None, None, *out)


class Rotary(torch.nn.Module):
    """Rotary positions: pair i of a head's values is turned by ``position * f_i`` radians,
    ``f_i = base ** (-2 i / rotary_dim)`` before scaling.

    Args:
        head_dim: values of a head, at most 512.
        rotary_dim: how many of them turn, from the first on (even; ``None``: all).
        base: of the frequencies.
        interleaved: pairs are ``(2 i, 2 i + 1)``; else ``(i, i + rotary_dim / 2)``.
        scaling: for contexts longer than the trained one, a dict with a ``type``:
            ``"linear"``: all frequencies by ``1 / factor``;
            ``"ntk"``: ``base`` by ``factor ** (rotary_dim / (rotary_dim - 2))``;
            ``"yarn"``: pairs that turn more than ``beta_fast`` (32) times in
            ``original_length`` positions stay, those below ``beta_slow`` (1) go by ``1 /
            factor``, a ramp over the pairs between; the result by ``amplitude`` (``0.1
            ln(factor) + 1``);
            ``"bands"``: pairs above ``high`` (4) turns in ``original_length`` positions stay,
            those below ``low`` (1) go by ``1 / factor``, interpolated over the turns between.

    ``rotary(q, k, positions)`` turns two tensors ``[B, H, N, D]`` (heads of their own; bf16,
    fp16 or fp32; any strides) in one launch and returns them in the same layout (contiguous
    where rows overlap); ``rotary(q, positions=..)`` one. positions: int32 ``[N]`` or ``[B, N]`` on the
    device, any value (int64 is converted: past 32 bits the nearest one); ``None``: 0 .. N - 1. Angles are
    reduced to a turn within 2e-9 radians at every position (64-bit fixed point, no table), and what is left
    after quarter turns, up to pi / 4, is held in fp32 (1.5e-7 in all); the products are formed in fp32 and
    rounded once. ``B * N < 2**24``.

    Gradients of any order are recorded. A backward pass that is captured into a graph takes
    them with ``torch.autograd.grad``: leaves that an eager pass has accumulated gradients
    into belong to that pass's stream, whatever the operator.

    The frequencies are a buffer that goes to the module's device and is no part of its
    state dict; they are formed anew where it is (``to_empty`` after a start on the meta device).
    """

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0,
                 interleaved: bool = False, scaling: Optional[dict] = None):
        super().__init__()
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if not 2 <= self.rotary_dim <= self.head_dim <= 512 or self.rotary_dim % 2:
            raise ValueError("rotary_dim must be even, in [2, head_dim], and head_dim at most 512; got "
                             f"{self.rotary_dim} of {self.head_dim}")
        self.base = float(base)
        if not (math.isfinite(self.base) and self.base > 1.0):
            raise ValueError(f"base must be above 1; got {base}")
        self.interleaved = bool(interleaved)
        self.scaling = dict(scaling) if scaling else None
        self.frequencies, self.amplitude = _frequencies(self.rotary_dim, self.base, self.scaling)
        self.register_buffer("turns", self._formed(), persistent=False)

    def _formed(self) -> torch.Tensor:
        return torch.tensor([_turns(x) for x in self.frequencies], dtype=torch.int64)

    def reset_parameters(self) -> None:
        """Forms the buffer's values anew, where it lies."""
        with torch.device("cpu"):
            turns = self._formed()
        with torch.no_grad():
            self.turns.copy_(turns)

    def _apply(self, fn, *args, **kwargs):
        """(a buffer that is made anew, by ``to_empty`` say, would hold whatever the memory did: no state dict has
        its values)"""
        before = self.turns
        super()._apply(fn, *args, **kwargs)
        if self.turns is not before and not self.turns.is_meta and self.turns.dtype is torch.int64:
            self.reset_parameters()
        return self

    def extra_repr(self) -> str:
        return (f"head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, base={self.base}, "
                f"interleaved={self.interleaved}, scaling={self.scaling}")

    def plan(self):
        """``((rotary_dim, interleaved, amplitude), turns)``, what the kernels take."""
        turns = self.turns
        if turns.dtype is not torch.int64 or turns.numel() != self.rotary_dim // 2:
            raise RuntimeError("Rotary: the turns buffer has been converted; make a new module")
        return (self.rotary_dim, self.interleaved, self.amplitude), turns

    def forward(self, q: torch.Tensor, k: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None):
        tensors = (q,) if k is None else (q, k)
        for x in tensors:
            if x.dim() != 4 or x.shape[3] != self.head_dim:
                raise ValueError(f"expected [B, H, N, {self.head_dim}]; got {list(x.shape)}")
            if (x.shape[0], x.shape[2]) != (q.shape[0], q.shape[2]):
                raise ValueError("q and k must share B and N")
            if x.dtype is not q.dtype:
                raise TypeError("q and k dtypes differ")
        nat.dtype_code(q)
        plan, turns = self.plan()
        given = (*tensors, turns) if positions is None else (*tensors, turns, positions)
        record = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
        (_plain if record else nat.plain_index)("Rotary", *given)
        if positions is not None:
            B, N = q.shape[0], q.shape[2]
            positions = nat.index32(positions, "positions", (N,) if positions.dim() == 1 else (B, N))
        if record:
            out = _Turned.apply(plan, turns, positions, False, *tensors)
        else:
            out = _turn(plan, turns, positions, False, tensors)
        return out[0] if k is None else (out[0], out[1])
