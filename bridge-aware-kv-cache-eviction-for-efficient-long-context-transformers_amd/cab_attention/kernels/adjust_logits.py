"""Logits before the next token is chosen (``cab_adjust_logits``): penalties for repeated
tokens, biases and grammar masks in one pass. The reference samples nothing and has no
counterpart."""

from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _native as nat


def _penalty(x, name: str, logits: torch.Tensor):
    """``(array or None, value)`` of a penalty: fp32 ``[B]``, or one number for all."""
    if not isinstance(x, torch.Tensor):
        return None, float(x)
    B = logits.shape[0]
    if x.shape != (B,) or x.dtype is not torch.float32:
        raise ValueError(f"{name} must be a number or fp32 [{B}]; got {x.dtype} {list(x.shape)}")
    return x.contiguous(), 0.0


def adjust_logits(logits: torch.Tensor, history: Optional[torch.Tensor] = None,
                  lengths: Optional[torch.Tensor] = None,
                  prompt_lengths: Optional[torch.Tensor] = None,
                  repetition: Union[float, torch.Tensor] = 1.0,
                  presence: Union[float, torch.Tensor] = 0.0,
                  frequency: Union[float, torch.Tensor] = 0.0,
                  bias_tokens: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                  allowed: Optional[torch.Tensor] = None, drafts: Optional[torch.Tensor] = None,
                  parents: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits that :func:`verify_drafts` takes (with T = 1 it is a sampler), from the
    model's. With ``c`` the times a token was generated, in this order::

        seen before:  x = x / repetition if x > 0 else x * repetition
        c > 0:        x = x - frequency * c - presence
        a bias:       x = x + bias
        not allowed:  x = -inf

    Args:
        logits: ``[B, T, V]`` (bf16, fp16 or fp32), after one token a sequence (T = 1) or after
            each node of a tree of drafts.
        history: int32 ``[B, L]`` (int64 is converted), each sequence's tokens; those from
            ``lengths[b]`` on are not read (``None``: all L), those before
            ``prompt_lengths[b]`` (``None``: 0) are the prompt, which counts as seen but not as
            generated. Tokens outside the vocabulary count for nothing.
        repetition, presence, frequency: one number for all, or fp32 ``[B]`` on the device.
            repetition is positive.
        bias_tokens, bias: int32 (int64 is converted) and fp32, ``[B, n]``, the biases of n
            tokens a sequence. Entries outside the vocabulary are none; of a token that is listed
            twice the last one counts.
        allowed: int32 ``[B, W]`` or ``[B, T, W]``, ``W = ceil(V / 32)``: bit ``v % 32`` of word
            ``v // 32`` is set if token v may follow. ``None``: all may.
        drafts, parents: the tree's tokens ``[B, T]`` and parents ``[T]`` or ``[B, T]``, as
            :func:`verify_drafts` takes them: the tokens from a node up to its root (its own
            included) count as generated for its logits, so ``history`` ends before node 0's
            token. T <= 256.
        out: where the result goes, like logits; the logits themselves, or memory of none of the
            inputs.

    All arithmetic is in fp32, rounded once; values of which nothing is asked pass unchanged (a NaN
    as a NaN).
    """
    if logits.dim() != 3:
        raise ValueError(f"logits must be [B, T, V]; got {list(logits.shape)}")
    B, T, V = logits.shape
    given = [logits]
    for x in (history, lengths, prompt_lengths, repetition, presence, frequency, bias_tokens, bias,
              allowed, drafts, parents, out):
        if x is not None and not isinstance(x, (float, int)):
            given.append(x)
    dev = nat.plain_index("adjust_logits", *given)
    dt = nat.dtype_code(logits)
    L = history_ld = 0
    if history is not None:
        history, L, history_ld = nat.table32(history, "history", B)
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("lengths and prompt_lengths are the history's")
    if lengths is not None:
        lengths = nat.index32(lengths, "lengths", (B,))
    if prompt_lengths is not None:
        prompt_lengths = nat.index32(prompt_lengths, "prompt_lengths", (B,))
    repetition, repetition0 = _penalty(repetition, "repetition", logits)
    presence, presence0 = _penalty(presence, "presence", logits)
    frequency, frequency0 = _penalty(frequency, "frequency", logits)
    if (bias_tokens is None) != (bias is None):
        raise ValueError("bias_tokens and bias come together")
    n = bias_ld = 0
    if bias is not None:
        if bias.dim() != 2 or bias.shape[0] != B or bias.dtype is not torch.float32:
            raise ValueError(f"bias must be fp32 [{B}, n]; got {bias.dtype} {list(bias.shape)}")
        n = bias_ld = bias.shape[1]
        bias_tokens, bias = nat.index32(bias_tokens, "bias_tokens", (B, n)), bias.contiguous()
    allowed_strides = None
    if allowed is not None:
        W = -(-V // 32)
        if allowed.dtype is not torch.int32:
            raise TypeError(f"allowed must be int32 words of 32 bits; got {allowed.dtype}")
        if allowed.shape != (B, W) and allowed.shape != (B, T, W):
            raise ValueError(f"allowed must be {[B, W]} or {[B, T, W]}; got {list(allowed.shape)}")
        if allowed.stride(-1) != 1:
            allowed = allowed.contiguous()
        allowed_strides = nat.stride_array(
            (allowed.stride(0), 0 if allowed.dim() == 2 else allowed.stride(1)))
    if (drafts is None) != (parents is None):
        raise ValueError("drafts and parents come together")
    shared = True
    if drafts is not None:
        if drafts.shape != (B, T):
            raise ValueError(f"drafts must be {[B, T]}; got {list(drafts.shape)}")
        if drafts.dtype is not torch.int64:
            if drafts.dtype is not torch.int32:
                raise TypeError(f"drafts must be int64 or int32; got {drafts.dtype}")
            drafts = drafts.to(torch.int64)
        drafts = drafts.contiguous()
        shared = parents.dim() == 1
        parents = nat.index32(parents, "parents", (T,) if shared else (B, T))
    if out is not None:
        if out.shape != logits.shape or out.dtype is not logits.dtype:
            raise ValueError("out must match the logits' shape and dtype")
        if V > 1 and out.stride(2) != 1:
            raise ValueError("out needs a contiguous last dim")
        if nat.closed(out):
            raise RuntimeError("adjust_logits: out is an inference tensor; write to it in "
                               "inference mode")
    if logits.stride(2) != 1:
        logits = logits.contiguous()
    if out is None:
        out = logits.new_empty((B, T, V))
    else:
        nat.wrote(out)
    with nat.at_index(dev):
        st = nat.load().cab_adjust_logits(
            logits.data_ptr(), out.data_ptr(), dt, B, T, V, nat.stride_array(logits.stride()[:2]),
            nat.stride_array(out.stride()[:2]), nat.ptr(history), L, history_ld, nat.ptr(lengths),
            nat.ptr(prompt_lengths), nat.ptr(repetition), repetition0, nat.ptr(presence), presence0,
            nat.ptr(frequency), frequency0, nat.ptr(bias_tokens), nat.ptr(bias), n, bias_ld,
            nat.ptr(allowed), allowed_strides, nat.ptr(drafts), nat.ptr(parents), 0 if shared else T,
            nat.raw_stream(dev))
    if st:
        nat.check("cab_adjust_logits", st)
    return out
