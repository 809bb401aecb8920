"""Verification of drafted tokens (``cab_verify_drafts``): which path of a tree of
drafts the target model's own sampling would have taken, and the token after it.
The reference decodes one token at a time and has no counterpart."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native as nat


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor,
                  uniforms: Optional[torch.Tensor] = None, noise: Optional[torch.Tensor] = None,
                  temperature: float = 1.0, draft_logits: Optional[torch.Tensor] = None
                  ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Walks each sequence's tree from node 0 (the token the model has taken already)
    to the first child that is accepted, and so on; where none is, draws the next token
    from what the rejections left.

    Args:
        logits: ``[B, T, V]``, the target's after each node (bf16, fp16 or fp32).
        tokens: ``[B, T]``, the drafted tokens (node 0's is not read).
        parents: ``[T]`` or ``[B, T]``, each node's parent, below its own index. Nodes
            with a negative parent are nobody's children (a padded tree: -2). T <= 256.
        uniforms: fp32 ``[B, T]`` in [0, 1), one number per draft.
        noise: fp32 ``[B, V]``, ``torch.empty(B, V).exponential_()``: the next token is
            ``argmax(w / noise)``, a sample of the weights ``w``.
        temperature: of both models' softmax. 0 is greedy: a draft is accepted if it is
            the target's argmax, and uniforms, noise and draft_logits are not read.
        draft_logits: ``[B, T, V]`` like ``logits``: node i's children were drawn
            independently from their softmax, and are accepted or rejected so that the
            output is distributed as the target's samples. ``None``: the children are
            distinct candidates (the draft's likeliest, say), each accepted with the
            target's probability of it, given that its earlier siblings were not.

    Returns ``(path, counts, next_tokens)``: int32 ``[B, T]``, the accepted nodes,
    ascending from 0 and filled with -1; int32 ``[B]``, how many; int64 ``[B]``. Equal
    values go to the lowest index. A NaN logit weighs nothing. A row without any weight
    accepts no child, and gives the next token -1.
    """
    if logits.dim() != 3:
        raise ValueError(f"logits must be [B, T, V]; got {list(logits.shape)}")
    B, T, V = logits.shape
    dev = nat.plain_index("verify_drafts", logits, tokens, parents)
    dt = nat.dtype_code(logits)
    if tokens.shape != (B, T):
        raise ValueError(f"tokens must be {[B, T]}; got {list(tokens.shape)}")
    if tokens.dtype is not torch.int64:
        if tokens.dtype is not torch.int32:
            raise TypeError(f"tokens must be int64 or int32; got {tokens.dtype}")
        tokens = tokens.to(torch.int64)
    tokens = tokens.contiguous()
    shared = parents.dim() == 1
    parents = nat.index32(parents, "parents", (T,) if shared else (B, T))
    temperature = float(temperature)
    if temperature == 0.0:
        uniforms = noise = draft_logits = None
    else:
        if uniforms is None or noise is None:
            raise ValueError("sampling (temperature > 0) needs uniforms and noise")
        nat.plain_index("verify_drafts", logits, uniforms, noise)
        for t, name, shape in ((uniforms, "uniforms", (B, T)), (noise, "noise", (B, V))):
            if t.shape != shape or t.dtype is not torch.float32:
                raise ValueError(f"{name} must be fp32 {list(shape)}; got {t.dtype} {list(t.shape)}")
        uniforms, noise = uniforms.contiguous(), noise.contiguous()
    if logits.stride(2) != 1:
        logits = logits.contiguous()
    ls = ds = nat.stride_array(logits.stride()[:2])
    if draft_logits is not None:
        if draft_logits.shape != logits.shape or draft_logits.dtype is not logits.dtype:
            raise ValueError("draft_logits must match logits' shape and dtype")
        nat.plain_index("verify_drafts", logits, draft_logits)
        if draft_logits.stride(2) != 1:
            draft_logits = draft_logits.contiguous()
        ds = nat.stride_array(draft_logits.stride()[:2])
    lib = nat.load()
    wbytes = lib.cab_verify_drafts_workspace_bytes(dt, B, T, V, temperature == 0.0,
                                                   draft_logits is not None)
    ws = logits.new_empty(wbytes, dtype=torch.uint8) if wbytes else None
    path = parents.new_empty((B, T))
    counts = parents.new_empty(B)
    chosen = tokens.new_empty(B)
    with nat.at_index(dev):
        st = lib.cab_verify_drafts(
            logits.data_ptr(), nat.ptr(draft_logits), dt, B, T, V, ls, ds, tokens.data_ptr(),
            parents.data_ptr(), 0 if shared else T, nat.ptr(uniforms), nat.ptr(noise), temperature,
            path.data_ptr(), counts.data_ptr(), chosen.data_ptr(), nat.ptr(ws), wbytes,
            nat.raw_stream(dev))
    if st:
        nat.check("cab_verify_drafts", st)
    return path, counts, chosen
