"""Attention of a tree of drafted tokens over a cache (``cab_tree_attn_fwd``), and of one
token a sequence over caches with lengths of their own (a tree of one node). The
reference decodes one token at a time over one length and has no counterpart."""

from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _native as nat


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, parents: torch.Tensor,
                   lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """``softmax(q k^T * scale) v`` over the keys each node sees: the sequence's context,
    and of the drafts behind it the node itself and its ancestors.

    Args:
        q: ``[B, H, T, D]``, the T nodes' queries; D = 64 or 128; bf16, fp16 or fp32.
        k, v: ``[B, H_kv, N, D]``, the cache, ``H % H_kv == 0`` (query head h reads head
            ``h // (H // H_kv)``). Sequence b's context is rows ``[0, lengths[b])``, its
            drafts the next T rows (see ``cache.append_drafts``); rows behind them are not
            read.
        parents: ``[T]`` or ``[B, T]`` int32: -1 for a node that hangs on the context
            alone, else an earlier node. Any other value means no node: it and what hangs
            on it see nothing (output 0, lse -inf), and nobody sees them. T <= 256.
        lengths: int32 ``[B]`` on the device, in ``[0, N - T]`` (others count as the
            nearest one inside). ``None``: the drafts are the last T rows.
        scale: defaults to ``1/sqrt(D)``.
        out: where the output goes, like q; q itself, or memory of none of the inputs.

    What a node does not see cannot reach its output, not even as a NaN or an infinity.
    A node that is there and whose scores have no softmax (a NaN or +inf among them, or
    all -inf) has NaN for its output and its log-sum-exp.
    Returns the output ``[B, H, T, D]``, with ``return_lse`` also the fp32 natural-log
    log-sum-exp ``[B, H, T]``.
    """
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q, k and v must be [B, H, T, D] and two [B, H_kv, N, D]")
    B, H, T, D = q.shape
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"k and v must be [B={B}, H_kv, N, D={D}]; got {list(k.shape)}")
    if not (q.dtype is k.dtype is v.dtype):
        raise TypeError("q, k, v dtypes differ")
    H_kv, N = k.shape[1], k.shape[2]
    if lengths is None:
        dev = nat.plain_index("tree_attention", q, k, v, parents)
    else:
        dev = nat.plain_index("tree_attention", q, k, v, parents, lengths)
        lengths = nat.index32(lengths, "lengths", (B,))
    dt = nat.dtype_code(q)
    shared = parents.dim() == 1
    parents = nat.index32(parents, "parents", (T,) if shared else (B, T))
    if out is None:
        out = q.new_empty((B, H, T, D))
    else:
        if out.shape != q.shape or out.dtype is not q.dtype:
            raise ValueError("out must match q's shape and dtype")
        nat.plain_index("tree_attention", q, out)
        if nat.closed(out):
            raise RuntimeError("tree_attention: out is an inference tensor; write to it in "
                               "inference mode")
        nat.wrote(out)
    q, k, v = nat.aligned_rows(q), nat.aligned_rows(k), nat.aligned_rows(v)
    lse = q.new_empty((B, H, T), dtype=torch.float32) if return_lse else None
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    lib = nat.load()
    arr = nat.stride_array
    wbytes = lib.cab_tree_attn_workspace_bytes(dt, B, H, H_kv, T, N, D)
    ws = q.new_empty(wbytes or 16, dtype=torch.uint8)
    with nat.at_index(dev):
        st = lib.cab_tree_attn_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, B, H, H_kv, T, N, D, arr(q.stride()),
            arr(k.stride()), arr(v.stride()), arr(out.stride()), parents.data_ptr(),
            0 if shared else T, nat.ptr(lengths), 0 if lengths is not None else N - T, scale, out.data_ptr(), nat.ptr(lse), ws.data_ptr(),
            wbytes, nat.raw_stream(dev))
    if st:
        nat.check("cab_tree_attn_fwd", st)
    return (out, lse) if return_lse else out
