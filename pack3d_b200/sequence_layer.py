"""Attention over ordered sequences as a layer on the residual stream, beside :class:`~pack3d_b200.FeedForward`.

:class:`SequenceAttention` runs :func:`~pack3d_b200.norm`, its projections, :func:`~pack3d_b200.norm_rotate`,
:func:`~pack3d_b200.sequence_attention` (or a :class:`~pack3d_b200.PagedCache` and :func:`~pack3d_b200.paged_attention`) and
:func:`~pack3d_b200.residual_norm` together.  No counterpart in the reference, whose layer attends over a geometry
(``src/pack3d/attention.py:12-89``).
"""
import math

import torch
from torch import nn

from .cache import PagedCache, paged_attention
from .residual import NormSpec, norm, residual_norm
from .sequence import norm_rotate, sequence_attention


class SequenceAttention(nn.Module):
    """``x + to_out(attention(norm_rotate(q), norm_rotate(k), v))``, ``q, k, v = to_qkv(pre_norm(x))``, within each sequence.

    Input / output ``[rows, dim]``, sequences one behind the other (``offsets`` as for :func:`sequence_attention`), fp16 or bf16
    on a CUDA sm_100 device.  ``positions`` [rows] or [rows, axes] as for :func:`norm_rotate`; queries and keys are RMS-normalised
    for each head unless ``head_norm=False``.  A stack hands the norm on as :class:`FeedForward` does: ``normed`` is the
    ``pre_norm`` of x that the block before made, and ``next_norm`` that of the block behind.

    For serving, :meth:`prefill` runs a prompt and writes its keys and values into a cache, :meth:`decode` one more token of
    each sequence.  Both read and write the cache behind ``lengths`` tokens and leave advancing them to the caller, so that
    a stack of layers shares them::

        cache = layer.new_cache(pages=1024, page_size=64, dtype=torch.float8_e4m3fn)
        with torch.no_grad():
            out, _ = layer.prefill(x, positions, offsets, cache, table, lengths)
            lengths += offsets.diff()
            out, _ = layer.decode(token, lengths, cache, table, lengths)
            lengths += 1
    """

    def __init__(self, dim, *, heads, kv_heads, head_dim, norm="rms", eps=1e-6, head_norm=True, causal=True, base=10000.0):
        super().__init__()
        if any(type(v) is not int or v <= 0 for v in (dim, heads, kv_heads, head_dim)):
            raise ValueError("dimensions must be positive integers")
        if heads % kv_heads:
            raise ValueError("query heads must be divisible by KV heads")
        if head_dim % 8 or head_dim > 128:
            raise ValueError("head_dim must be a multiple of 8 up to 128")
        if norm not in ("layer", "rms"):
            raise ValueError("norm must be layer or rms")
        self.dim, self.heads, self.kv_heads, self.head_dim = dim, heads, kv_heads, head_dim
        self.kind, self.eps, self.causal, self.base = norm, float(eps), bool(causal), float(base)
        self.pre_weight = nn.Parameter(torch.ones(dim))
        self.pre_bias = nn.Parameter(torch.zeros(dim)) if norm == "layer" else None
        self.q_weight = nn.Parameter(torch.ones(head_dim)) if head_norm else None
        self.k_weight = nn.Parameter(torch.ones(head_dim)) if head_norm else None
        self.to_qkv = nn.Linear(dim, (heads + 2 * kv_heads) * head_dim, bias=False)
        self.to_out = nn.Linear(heads * head_dim, dim, bias=False)

    @property
    def pre_norm(self):
        """The norm before the layer, for the ``next_norm`` of the block before it."""
        return NormSpec(self.pre_weight, self.pre_bias, self.kind, self.eps)

    def new_cache(self, pages, page_size, *, dtype=None, device=None):
        """A :class:`PagedCache` for this layer's keys and values (default: the parameters' dtype and device)."""
        weight = self.to_qkv.weight
        return PagedCache(pages, self.kv_heads, page_size, self.head_dim, dtype=dtype or weight.dtype, device=device or weight.device)

    def _qkv(self, x, positions, normed):
        if x.ndim != 2 or x.shape[1] != self.dim:
            raise ValueError(f"x must be [rows, {self.dim}], got {list(x.shape)}")
        y = norm(x, self.pre_norm) if normed is None else normed
        row = self.to_qkv(y)
        h, g, d = self.heads, self.kv_heads, self.head_dim
        q, k, v = row.split((h * d, g * d, g * d), -1)
        specs = (None, None) if self.q_weight is None else (NormSpec(w, None, "rms", self.eps) for w in (self.q_weight, self.k_weight))
        q_norm, k_norm = specs
        q, k = norm_rotate(q.unflatten(-1, (h, d)), k.unflatten(-1, (g, d)), positions, q_norm=q_norm, k_norm=k_norm, base=self.base)
        return q, k, v.unflatten(-1, (g, d))

    def _out(self, x, a, next_norm):
        return residual_norm(x, self.to_out(a.flatten(-2)), next_norm=next_norm)

    def forward(self, x, positions, offsets, *, normed=None, next_norm=None):
        """``(out, next_norm(out))``, the second None without ``next_norm``."""
        q, k, v = self._qkv(x, positions, normed)
        return self._out(x, sequence_attention(q, k, v, offsets, causal=self.causal), next_norm)

    def prefill(self, x, positions, offsets, cache, table, lengths, *, cached_rows=None, normed=None, next_norm=None):
        """:meth:`forward` for the new tokens of each sequence, which go into the cache behind ``lengths`` [sequences] tokens.

        ``cached_rows``: the number of tokens that all sequences have with these, where any had some before: keys and values are
        then read back from the cache (as it holds them, the new ones too).  Without it the sequences that have new tokens
        have to begin with them: where one of those has a length, its first tokens would be missing, and all results are
        NaN.  No gradients.
        """
        q, k, v = self._qkv(x, positions, normed)
        cache.append(k, v, table, lengths, offsets)
        if cached_rows is None:
            a = sequence_attention(q, k, v, offsets, causal=self.causal)
            # lengths are on the device: a refusal would wait for it
            a.masked_fill_(((lengths != 0) & (offsets.diff() != 0)).any(), math.nan)
        else:
            all_offsets = torch.nn.functional.pad((lengths + offsets.diff()).cumsum(0, dtype=torch.int32), (1, 0))
            k, v = cache.read(table, all_offsets, cached_rows, dtype=q.dtype)
            a = sequence_attention(q, k, v, offsets, all_offsets, causal=self.causal)
        return self._out(x, a, next_norm)

    def decode(self, x, positions, cache, table, lengths, *, normed=None, next_norm=None):
        """One more token of each sequence: row b of ``x`` [sequences, dim] goes into the cache as token ``lengths[b]`` of sequence b and
        attends to all of that sequence's.  No gradients; may be captured in a CUDA graph."""
        q, k, v = self._qkv(x, positions, normed)
        cache.append(k, v, table, lengths, torch.arange(x.shape[0] + 1, dtype=torch.int32, device=x.device))
        return self._out(x, paged_attention(q, cache, table, lengths + 1), next_norm)


__all__ = ["SequenceAttention"]
