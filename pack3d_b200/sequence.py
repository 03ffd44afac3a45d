"""Attention over ordered sequences of tokens: prompts, documents, autoregressive orders of a volume.

* :func:`norm_rotate` -- norms of queries and keys for each head and the rotation of their positions, one kernel a direction.
* :func:`sequence_attention` -- attention over sequences packed one behind the other, grouped heads, both directions.

Steps of both may be captured in CUDA graphs; a leaf that a living graph from the default stream still holds is refused there.

For serving, :mod:`pack3d_b200.cache` keeps keys and values in pages.  No counterpart in the reference, whose attention is
over a geometry (``reference.py:8-31``) and whose rotation stands alone (``rope.py:15-48``).
"""
from __future__ import annotations

from . import _native


def norm_rotate(q, k, positions, *, q_norm=None, k_norm=None, pairs=None, base=10000.0):
    """``(q', k')``: each head of ``q`` [.., tokens, heads, head_dim] and ``k`` [.., tokens, kv_heads, head_dim] (or None)
    normalised by its :class:`~pack3d_b200.NormSpec` (``q_norm``, ``k_norm``; None: not at all) over head_dim, then rotated.

    ``positions``: int32 or int64, [tokens], or [tokens, axes] for up to three axes, shared by the leading dimensions.  The
    axes own the pairs of columns (2 i, 2 i + 1) in turn, ``pairs`` of them each (default: all of them, dealt evenly, as
    :func:`~pack3d_b200.balanced_pairs`); columns past the last pair are not rotated.  Pair i of n of an axis turns by
    ``position * base**(-i / n)`` radians.  A frequency is that power in fp64, to 2^-64 turns, and its product with the position
    is exact, unlike in :func:`~pack3d_b200.rotate_projections`, which has the reference's fp32 angles bit for bit.

    fp32, fp16 or bf16, an even head_dim up to 256, any strides; statistics in fp32, one rounding at the end.  Results are
    contiguous.  Differentiable once in q, k and the norms' parameters, whose gradients are summed in fp32 in a fixed
    order; second and forward-mode derivatives are refused.
    """
    return _native.host().norm_rotate(q, k, positions, q_norm, k_norm, pairs, base)


def sequence_attention(q, k, v, q_offsets, k_offsets=None, *, causal=True, scale=None):
    """``softmax(scale q k^T) v`` within each sequence, [rows, heads, head_dim].

    ``q`` [rows, heads, head_dim], ``k`` and ``v`` [rows, kv_heads, head_dim] hold sequences one behind the other: sequence b is
    rows ``offsets[b]`` to ``offsets[b + 1]`` (int32 [sequences + 1] on the device, from 0 and not decreasing).  ``k_offsets``: the
    same for the keys, where they have other lengths (a cached prefix before the new tokens).  heads is a multiple of
    kv_heads; query head h reads KV head ``h // (heads // kv_heads)``.  With ``causal`` the last query of a sequence sees its
    last key, each query before it one key less.  ``scale``: default ``head_dim ** -0.5``.

    A query that sees no key gives 0 and sends no gradient, as do rows behind the last sequence, whatever they hold.  An
    infinity or NaN reaches the queries that see it and nothing else: no earlier query, no other sequence.  A query with a score
    of +inf, or with none but -inf, has no softmax: NaN.

    fp16 or bf16, head_dim a multiple of 8 up to 128; rows that are not 16-byte aligned are copied first.  Scores and sums in
    fp32; what goes into a product (weights, and score gradients from the rounded output) is rounded to the inputs' dtype, in
    fp16 times powers of two that bring it into range; exponentials are good to 2^-13.  Every sum has a fixed order, so the gradients are bitwise
    repeatable.  Differentiable once, in reverse mode; second and forward-mode derivatives are
    refused.
    """
    return _native.host().sequence_attention(q, k, v, q_offsets, k_offsets, causal, scale)


__all__ = ["norm_rotate", "sequence_attention"]
