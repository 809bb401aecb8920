"""Drafted tokens in K/V caches whose sequences have lengths of their own: new
rows written behind each sequence's length (``cab_kv_append_at``), and after
verification the accepted ones kept (``cab_kv_commit``). Lengths, counts and
paths stay on the device, so a decoding loop reads nothing back and can be
captured into a graph. The reference has neither: its caches hold one length and
grow by ``torch.cat`` (cache/cab_cache.py:122-175).

One step of a loop over static buffers ``[B, H_kv, N, D]`` per layer::

    for layer: append_drafts(k, v, keys[layer], values[layer], lengths)
               tree_attention(q, keys[layer], values[layer], parents, lengths)
    path, counts, token = verify_drafts(logits, tokens, parents, uniforms, noise)
    lengths = commit_drafts(keys + values, lengths, path, counts)
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence

import torch

from .. import _native as nat

_SIZES = {torch.bfloat16: 2, torch.float16: 2, torch.float32: 4}


@functools.lru_cache(maxsize=1024)
def _four_strides(*strides: tuple):
    return tuple(nat.stride_array(x) for x in strides)


def _writable(fn: str, *caches: torch.Tensor) -> None:
    for c in caches:
        if nat.closed(c):
            raise RuntimeError(f"{fn}: a cache is an inference tensor; write to it in inference mode")


def append_drafts(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  lengths: torch.Tensor, counts: Optional[torch.Tensor] = None) -> None:
    """``cache[b, :, lengths[b] + t] = new[b, :, t]`` for ``t < counts[b]``, K and V in
    one launch.

    k, v: ``[B, H, n, D]``, any strides. k_cache, v_cache: ``[B, H, N, D]`` of the same
    dtype (bf16, fp16, fp32) with a contiguous last dim. lengths, counts (``None``: n
    rows of every sequence): int32 ``[B]`` on the device (int64 is converted). Rows that
    would lie behind the cache's N, and those of a sequence of negative length, are
    not written. The new rows must not be views of the caches, nor
    the caches share memory.
    """
    new, shape = k.shape, k_cache.shape
    if len(new) != 4 or v.shape != new:
        raise ValueError("k and v must be two [B, H, n, D] tensors")
    B, H, n, D = new
    if len(shape) != 4 or v_cache.shape != shape or (shape[0], shape[1], shape[3]) != (B, H, D):
        raise ValueError(f"k_cache and v_cache must be [{B}, {H}, N, {D}]; got {tuple(shape)} and "
                         f"{tuple(v_cache.shape)}")
    dt = k.dtype
    es = _SIZES.get(dt)
    if es is None or v.dtype is not dt or k_cache.dtype is not dt or v_cache.dtype is not dt:
        raise TypeError("k, v and the caches must be of one dtype: bfloat16, float16 or float32")
    dev = nat.plain_index("append_drafts", k, v, k_cache, v_cache, lengths)
    if k_cache.is_inference() or v_cache.is_inference():
        _writable("append_drafts", k_cache, v_cache)
    lengths = nat.index32(lengths, "lengths", (B,))
    if counts is not None:
        nat.plain_index("append_drafts", k, counts)
        counts = nat.index32(counts, "counts", (B,))
    strides = _four_strides(k.stride(), v.stride(), k_cache.stride(), v_cache.stride())
    with nat.at_index(dev):
        st = nat.load().cab_kv_append_at(
            k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), es, B, H, n, D,
            shape[2], *strides, lengths.data_ptr(), nat.ptr(counts), nat.raw_stream(dev))
    if st:
        nat.check("cab_kv_append_at", st)
    nat.wrote(k_cache, v_cache)


def commit_drafts(caches: Sequence[torch.Tensor], lengths: torch.Tensor, path: torch.Tensor,
                  counts: torch.Tensor) -> torch.Tensor:
    """Keeps the accepted ones of each sequence's drafted rows, in every cache of the
    list (all layers' K and V, one launch per 64): row ``lengths[b] + path[b, j]``
    moves to row ``lengths[b] + j`` for ``j < counts[b]``. Returns the new lengths,
    int32 ``[B]``: the old ones plus the rows kept. No other row changes.

    caches: ``[B, H, N, D]`` tensors that share no memory, of one shape, dtype (bf16, fp16, fp32)
    and stride set, with a contiguous last dim. lengths, counts: int32 ``[B]``; path:
    int32 ``[B, T]``, on the device, as :func:`verify_drafts` gives them (int64 is
    converted). A path's first ``counts[b]`` entries ascend strictly; the first one
    that does not, or that lies outside ``[0, T)`` or the cache, ends it.
    """
    caches = list(caches)
    if not caches:
        raise ValueError("commit_drafts needs at least one cache")
    ref = caches[0]
    shape, stride, dt = ref.shape, ref.stride(), ref.dtype
    es = _SIZES.get(dt)
    if len(shape) != 4 or path.dim() != 2:
        raise ValueError("caches must be [B, H, N, D] and path [B, T]")
    if es is None:
        raise TypeError(f"unsupported dtype {dt}; expected float32, float16 or bfloat16")
    B = shape[0]
    alike, grad = ref.get_device(), torch.is_grad_enabled()
    for c in caches:  # (every layer's K and V: as few questions as there can be)
        if c.shape != shape or c.dtype is not dt or c.stride() != stride:
            raise ValueError("the caches must share one shape, dtype and stride set")
        if (type(c) is not torch.Tensor or c.get_device() != alike or c.is_inference()
                or (grad and c.requires_grad)):
            nat.plain_index("commit_drafts", ref, c)
            _writable("commit_drafts", c)
    dev = nat.plain_index("commit_drafts", ref, lengths, path, counts)
    lengths = nat.index32(lengths, "lengths", (B,))
    counts = nat.index32(counts, "counts", (B,))
    path = nat.index32(path, "path", (B, path.shape[1]))
    new = torch.empty_like(counts)
    _commit(caches, lengths, 0, path, counts, 0, new, dev, es)
    return new


def _commit(caches, lengths, length, path, counts, count, new, dev, es, columns=None):
    B, H, N, D = caches[0].shape
    n = len(caches)
    st = caches[0].stride()
    if columns is not None:  # rows as values of another size
        D, st = columns, tuple(x * columns // D for x in st[:3]) + (1,)
    ptrs = (ctypes.c_void_p * n)(*[c.data_ptr() for c in caches])
    with nat.at_index(dev):
        status = nat.load().cab_kv_commit(
            ptrs, n, es, B, H, N, D, nat.stride_array(st), nat.ptr(lengths), length, path.data_ptr(),
            path.shape[-1], path.shape[-1] if path.dim() == 2 else 0, nat.ptr(counts), count,
            nat.ptr(new), nat.raw_stream(dev))
    if status:
        nat.check("cab_kv_commit", status)
    nat.wrote(*caches)


def commit_rows(groups: Sequence[tuple], count: int) -> None:
    """:func:`commit_drafts` for groups ``(caches, path, length)`` of contiguous buffers of
    one shape and length, ``length`` rows before the drafts, of which every sequence keeps
    ``count`` (int32 path ``[B, T]``, or ``[T]`` for all). Rows of any dtype whose bytes are
    a multiple of 4. All groups are checked before the first row moves."""
    devs = []
    for caches, path, _ in groups:
        devs.append(nat.plain_index("commit", path, *caches))
        _writable("commit", *caches)
        if caches[0].shape[0] > 65535 or len(caches) > 4096:
            raise ValueError("commit takes up to 65535 sequences and 2048 layers of one geometry")
    for (caches, path, length), dev in zip(groups, devs):
        ref = caches[0]
        _commit(caches, None, length, path, None, count, None, dev, 4,
                ref.shape[3] * ref.element_size() // 4)
