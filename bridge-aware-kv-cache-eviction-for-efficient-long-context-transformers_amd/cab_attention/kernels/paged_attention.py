"""Attention of one token a sequence over a cache in pages (``cab_paged_attn_fwd``). The
reference decodes over caches of one length that lie in one piece, and has no counterpart."""

from __future__ import annotations

import functools
import math
from typing import Optional

import torch

from .. import _native as nat


@functools.lru_cache(maxsize=1024)
def _checked(q, kv, v, q_dtype, k_dtype, v_dtype):
    """``(B, H, D, P, H_kv, S)`` of the shapes, once for each set of them (a step of a decoding
    loop asks the same per layer)."""
    if len(q) != 4 or q[2] != 1 or len(kv) != 4 or v != kv:
        raise ValueError("q must be [B, H, 1, D], k_pages and v_pages two [P, H_kv, S, D]")
    if kv[3] != q[3]:
        raise ValueError(f"k_pages and v_pages must be [P, H_kv, S, D={q[3]}]; got {list(kv)}")
    if not (q_dtype is k_dtype is v_dtype):
        raise TypeError("q, k_pages and v_pages dtypes differ")
    return q[0], q[1], q[3], kv[0], kv[1], kv[2]


@functools.lru_cache(maxsize=1024)
def _layout(dt, sizes, columns, *strides):
    """The workspace's bytes and the strides as C integers."""
    B, H, D, _, H_kv, S = sizes
    need = nat.load().cab_paged_attn_workspace_bytes(dt, B, H, H_kv, columns, S, D)
    return need, tuple(nat.stride_array(x) for x in strides)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """``softmax(q k^T * scale) v`` over the first ``lengths[b]`` rows of each sequence, which
    lie in the pages that its row of the table names.

    Args:
        q: ``[B, H, 1, D]``, one token a sequence; D = 64 or 128; bf16, fp16 or fp32.
        k_pages, v_pages: ``[P, H_kv, S, D]``, P pages of S rows (any S; whole multiples of
            16 are fastest), ``H % H_kv == 0`` (query head h reads head ``h // (H // H_kv)``);
            any strides with a contiguous last dim and rows on 16-byte boundaries (a pool laid
            out ``[P, S, H_kv, D]`` goes in as its transposed view).
        page_table: int32 ``[B, M]`` on the device (int64 is converted): row s of sequence b is
            place ``s % S`` of page ``page_table[b, s // S]``. An entry outside ``[0, P)`` (-1,
            say) is no page: its rows are not seen (evicted, or never written). Sequences may
            share pages.
        lengths: int32 ``[B]`` on the device, the rows a sequence sees, its own token's
            included (see ``cache.append_paged``). Values outside ``[0, M S]`` count as the
            nearest one inside.
        scale: defaults to ``1/sqrt(D)``; positive, and below 2.3e38.
        out: where the output goes, like q; q itself, or memory of none of the inputs.

    Rows behind a length, and pages that are not the sequence's, are not read. A sequence that
    sees no row has output 0 and log-sum-exp -inf. One whose scores have no softmax (a NaN or
    +inf among them, or all -inf; ``q k^T`` past fp32's range is infinite) has NaN for both. Scores,
    weights, their sum and the sum of weights times values are held in fp32, relative to the largest
    weight (below 2^-126 of it a weight is 0; for the product with 16-bit values weights have 24 bits in
    bf16, 22 in fp16); the output is rounded once.
    Returns the output ``[B, H, 1, D]``, with ``return_lse`` also the fp32 natural-log
    log-sum-exp ``[B, H, 1]``.
    """
    sizes = _checked(q.shape, k_pages.shape, v_pages.shape, q.dtype, k_pages.dtype, v_pages.dtype)
    B, H, D, P, H_kv, S = sizes
    dev = nat.plain_index("paged_attention", q, k_pages, v_pages, page_table, lengths)
    dt = nat.dtype_code(q)
    page_table, M, ld = nat.table32(page_table, "page_table", B)
    lengths = nat.index32(lengths, "lengths", (B,))
    rows = nat.aligned_rows(q)
    if out is None:
        out = torch.empty_like(rows)
    else:
        if out.shape != q.shape or out.dtype is not q.dtype:
            raise ValueError("out must match q's shape and dtype")
        nat.plain_index("paged_attention", q, out)
        if nat.closed(out):
            raise RuntimeError("paged_attention: out is an inference tensor; write to it in "
                               "inference mode")
        nat.wrote(out)
    q = rows
    lse = q.new_empty((B, H, 1), dtype=torch.float32) if return_lse else None
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    wbytes, strides = _layout(dt, sizes, M, q.stride(), k_pages.stride(), v_pages.stride(),
                              out.stride())
    ws = q.new_empty(wbytes, dtype=torch.uint8) if wbytes else None
    with nat.at_index(dev):
        st = nat.load().cab_paged_attn_fwd(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), dt, B, H, H_kv, D, P, S,
            *strides, page_table.data_ptr(), ld, M, lengths.data_ptr(), scale, out.data_ptr(),
            nat.ptr(lse), nat.ptr(ws), wbytes, nat.raw_stream(dev))
    if st:
        nat.check("cab_paged_attn_fwd", st)
    return (out, lse) if return_lse else out
