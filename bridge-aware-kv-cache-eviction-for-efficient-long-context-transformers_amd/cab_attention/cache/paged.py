"""New rows in a cache that lies in pages (``cab_paged_append``): K rotated to its
positions on the way, the queries with it. Lengths and the page table stay on the device, so
a decoding loop reads nothing back and can be captured into a graph. The reference has
no pages: its caches grow by ``torch.cat`` (cache/cab_cache.py:122-175).

One step of a loop over pools ``[P, H_kv, S, D]`` per layer, one token a sequence::

    seen = lengths + 1
    for layer: q = append_paged(k, v, keys[layer], values[layer], table, lengths,
                                rotary=rotary, q=q)
               out = paged_attention(q, keys[layer], values[layer], table, seen)
    logits = adjust_logits(logits, history, seen, prompt_lengths, repetition=1.1)
    _, _, token = verify_drafts(logits, last_token, root, uniforms, noise)

A server that evicts takes a page out of the table (-1) and hands it on: attention no
longer sees its rows, and the others keep their positions.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _native as nat
from ..kernels.rotary import Rotary
from .drafts import _four_strides, _writable


def append_paged(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor,
                 counts: Optional[torch.Tensor] = None, rotary: Optional[Rotary] = None,
                 positions: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None
                 ) -> Optional[torch.Tensor]:
    """Row ``lengths[b] + t`` of sequence b becomes ``k[b, :, t]`` (rotated) and ``v[b, :, t]`` for
    ``t < counts[b]``: K, V and the queries in one launch.

    Args:
        k, v: ``[B, H_kv, n, D]``, any strides; bf16, fp16 or fp32; D <= 512, ``B * n < 2**24``.
        k_pages, v_pages: ``[P, H_kv, S, D]`` of the same dtype, contiguous in the last dim: row s
            of sequence b is place ``s % S`` of page ``page_table[b, s // S]``. They share
            no memory with each other or the new rows.
        page_table: int32 ``[B, M]`` on the device (int64 is converted). Rows past it, and those
            whose entry lies outside ``[0, P)``, are not written. A page that is written to
            belongs to one sequence: of rows that meet in one place, parts of either may stay.
        lengths, counts (``None``: n rows of every sequence): int32 ``[B]`` on the device. A
            sequence of negative length gets no row.
        rotary: turns k (and q); ``None``: k goes in as it is.
        positions: int32 ``[n]`` or ``[B, n]``, what ``rotary`` turns by; ``None``: the rows'
            own numbers, ``lengths[b] + t``. (A cache that has dropped rows has later positions.)
        q: ``[B, H, n, D]``, queries to be rotated to the same positions.

    Returns the rotated q (all n rows of it), or ``None`` without q.
    """
    new, shape = k.shape, k_pages.shape
    if len(new) != 4 or v.shape != new:
        raise ValueError("k and v must be two [B, H_kv, n, D] tensors")
    B, H_kv, n, D = new
    if len(shape) != 4 or v_pages.shape != shape or (shape[1], shape[3]) != (H_kv, D):
        raise ValueError(f"k_pages and v_pages must be [P, {H_kv}, S, {D}]; got {tuple(shape)} and "
                         f"{tuple(v_pages.shape)}")
    dt = k.dtype
    if v.dtype is not dt or k_pages.dtype is not dt or v_pages.dtype is not dt:
        raise TypeError("k, v and the pages must be of one dtype: bfloat16, float16 or float32")
    code = nat.dtype_code(k)
    given = [k, v, k_pages, v_pages, page_table, lengths]
    for x in (counts, positions, q):
        if x is not None:
            given.append(x)
    turns, plan, position_ld = None, (0, False, 1.0), 0
    if rotary is not None:
        plan, turns = rotary.plan()
        given.append(turns)
    dev = nat.plain_index("append_paged", *given)
    if k_pages.is_inference() or v_pages.is_inference():
        _writable("append_paged", k_pages, v_pages)
    page_table, M, ld = nat.table32(page_table, "page_table", B)
    lengths = nat.index32(lengths, "lengths", (B,))
    if counts is not None:
        counts = nat.index32(counts, "counts", (B,))
    if rotary is not None:
        if rotary.head_dim != D:
            raise ValueError(f"rotary is for heads of {rotary.head_dim} values; got {D}")
    elif q is not None or positions is not None:
        raise ValueError("q and positions are for rotary")
    if positions is not None:
        one = positions.dim() == 1
        positions = nat.index32(positions, "positions", (n,) if one else (B, n))
        position_ld = 0 if one else n
    H, out, q_strides, out_strides = 0, None, None, None
    if q is not None:
        if q.dim() != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (B, n, D):
            raise ValueError(f"q must be [{B}, H, {n}, {D}]; got {list(q.shape)}")
        if q.dtype is not dt:
            raise TypeError("q and k dtypes differ")
        if q.stride(3) != 1:
            q = q.contiguous()
        H, out = q.shape[1], nat.empty_rows_like(q)
        q_strides, out_strides = nat.stride_array(q.stride()), nat.stride_array(out.stride())
    if k.stride(3) != 1:
        k = k.contiguous()
    if v.stride(3) != 1:
        v = v.contiguous()
    strides = _four_strides(k.stride(), v.stride(), k_pages.stride(), v_pages.stride())
    with nat.at_index(dev):
        st = nat.load().cab_paged_append(
            k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), nat.ptr(q), nat.ptr(out),
            code, B, H, H_kv, n, D, shape[0], shape[2], *strides, q_strides, out_strides,
            page_table.data_ptr(), ld, M, lengths.data_ptr(), nat.ptr(counts), nat.ptr(positions),
            position_ld, nat.ptr(turns), *plan, nat.raw_stream(dev))
    if st:
        nat.check("cab_paged_append", st)
    nat.wrote(k_pages, v_pages)
    return out
