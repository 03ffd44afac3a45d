"""Keys and values of served sequences in pages, and the attention of a new token over them.

* :class:`PagedCache` -- pages in fp32, fp16, bf16 or in 8 bits with a power-of-two scale for each token and head;
  :meth:`~PagedCache.append` writes, :meth:`~PagedCache.read` reads back.
* :func:`paged_attention` -- one new token of each sequence over its pages.

A page table [sequences, width] of int32 says where a sequence's tokens are: token i in place ``i % page_size`` of page
``table[b, i // page_size]``.  Who gets which page is the caller's business; pages may be shared by sequences that read
them.  No counterpart in the reference, which attends over whole volumes (``attention.py:53-89``).
"""
from __future__ import annotations

import torch

from . import _native


class PagedCache:
    """``k`` and ``v`` [pages, kv_heads, page_size, head_dim] and, for ``dtype=torch.float8_e4m3fn``, ``k_scales`` and ``v_scales``
    uint8 [pages, kv_heads, page_size], bytes e + 127 of the 2^e that a token's values of one head are multiplied by (otherwise
    None).  head_dim is a multiple of 8 up to 256.  The pages start as zeros.

    Tables, lengths and offsets are int32 tensors on the cache's device and are read by the kernels: a captured graph
    follows their contents.  A page number outside the cache is never followed: the write is dropped, a read gives
    NaN, and bit 6 of ``p3d_device_errors`` is set.
    """

    __slots__ = ("k", "v", "k_scales", "v_scales")

    def __init__(self, pages, kv_heads, page_size, head_dim, *, dtype=torch.bfloat16, device="cuda"):
        for name, value in (("pages", pages), ("kv_heads", kv_heads), ("page_size", page_size), ("head_dim", head_dim)):
            if type(value) is not int or value < 1:
                raise ValueError(f"{name} must be a positive integer")
        if head_dim % 8 or head_dim > 256:
            raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {head_dim}")
        if dtype is not torch.float8_e4m3fn and dtype not in _native.DTYPE_CODE:
            raise ValueError("dtype must be fp32, fp16, bf16 or float8_e4m3fn")
        shape = (pages, kv_heads, page_size, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.k_scales = self.v_scales = None
        if dtype is torch.float8_e4m3fn:
            self.k_scales, self.v_scales = (torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2))

    @property
    def page_size(self):
        return self.k.shape[2]

    @property
    def dtype(self):
        return self.k.dtype

    @property
    def device(self):
        return self.k.device

    def append(self, k, v, table, lengths, offsets):
        """Write new tokens: row ``offsets[b] + i`` of ``k`` and ``v`` [rows, kv_heads, head_dim] becomes token ``lengths[b] + i`` of
        sequence b, for ``i < offsets[b + 1] - offsets[b]``.  Other rows are not read and other places stay as they are; the
        caller advances ``lengths``.  Into 8 bits each token and head is scaled by the smallest power of two that brings its
        largest finite magnitude to at most 448 and rounded to nearest even (infinities and NaN become NaN).  Two rows for
        one place leave a mixture of them.  No gradients."""
        _native.host().cache_append(self.k, self.v, self.k_scales, self.v_scales, table, k, v, lengths, offsets)

    def read(self, table, offsets, rows, *, starts=None, dtype=None):
        """``(k, v)`` [rows, kv_heads, head_dim] of ``dtype`` (default: the cache's, bf16 for 8 bits): row ``offsets[b] + i`` is token
        ``i`` (``starts[b] + i``) of sequence b.  ``rows`` is ``offsets[-1]`` as the caller knows it; rows of no sequence are 0."""
        return _native.host().cache_read(self.k, self.v, self.k_scales, self.v_scales, table, starts, offsets, rows, dtype)


def paged_attention(q, cache, table, lengths, *, scale=None):
    """``softmax(scale q k^T) v`` of one query of each sequence, ``q`` [sequences, heads, head_dim], over tokens 0 to ``lengths[b]`` of
    its pages (the new token's own among them, once appended); 0 for a sequence without any.

    fp16 or bf16 queries, of the cache's dtype where that is 16-bit, or any of the two over 8 bits; head_dim up to 128; heads
    a multiple of the cache's.  Scores and sums in fp32, weights rounded to the pages' 16-bit type; over 8 bits, which enter
    exactly, to fp16, as queries are relative to their largest column.  The same call gives the same bits: the order of a
    sum depends on the batch's lengths, the heads, the device, and on whether the table is wider than four units of 128 tokens
    (of 64, over 16-bit pages with a head_dim above 64), not on how much wider.  No gradients.
    """
    if not isinstance(cache, PagedCache):
        raise ValueError("paged_attention takes a PagedCache")
    return _native.host().paged_attention(cache.k, cache.v, cache.k_scales, cache.v_scales, table, q, lengths, scale)


__all__ = ["PagedCache", "paged_attention"]
