"""The parts of a transformer block around its matrix products: norms before and after the block with its gate,
dropout, residual scale and residual, and dropout by itself, each one kernel in each direction.

* :func:`norm` -- RMS or layer norm over the last dimension.
* :func:`residual_norm` -- ``out = x + scale * dropout(post_norm(h) * act(gate))`` and ``y = next_norm(out)``.
* :func:`dropout` -- counter-based: the mask is a function of (seed, offset) and the element's place, made again in the
  backward pass and never stored.

No counterpart in the reference, whose layer ends at its own residual (``attention.py:89``).  fp32, fp16 and bf16 CUDA
tensors, any leading shape, up to 16,384 columns; statistics, sums and gradients of parameters in fp32, each value
rounded once where it is stored.  Differentiable once, in reverse mode; second and forward-mode derivatives are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native

MAX_DIM = 16384


class NormSpec(NamedTuple):
    """A norm over the last dimension: ``kind`` ``"rms"`` (``z / sqrt(mean(z^2) + eps)``) or ``"layer"``
    (``(z - mean) / sqrt(var + eps)``), times ``weight`` plus ``bias`` (either may be None)."""
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    kind: str = "rms"
    eps: float = 1e-6


def dropout(x, p, rng):
    """``x`` with each element zeroed with probability ``p`` and the others divided by ``1 - p``.

    ``rng`` is ``(seed, offset)``: two Python integers (64 bits are used), or a CUDA int64 tensor of the two, read
    by the kernel, for captured graphs (do not change it between the forward and the backward pass).  An
    element's fate depends on them and its place alone: with ``C`` columns, element ``(r, c)`` of the flattened
    rows is kept where 16-bit field ``c % 8`` of the Philox-4x32-10 block at counter ``(r * ceil(C / 8) + c // 8,
    offset)`` under key ``seed`` is at least ``T = round(65536 p)``; the scale is ``65536 / (65536 - T)``.  So a call
    uses up the offset it was given: take another for the next call.  The same mask as :func:`residual_norm`
    with the same ``rng`` and shape.
    """
    return _native.host().dropout(x, p, rng)


def norm(x, spec):
    """``spec`` (:class:`NormSpec`) of ``x`` over its last dimension, differentiable in ``x``, weight and bias."""
    return _native.host().norm(x, spec)


def residual_norm(x, h, *, post_norm=None, gate=None, gate_activation="identity", scale=None, next_norm=None, p=0.0,
                  rng=None):
    """The end of a block and the norm of the next one, in one kernel.

        u   = post_norm(h)                      (h, without post_norm)
        out = x + scale * dropout(u * act(gate), p)
        y   = next_norm(out)                    (None, without next_norm)

    ``x`` is the residual stream, ``h`` the block's output (same shape and dtype).  ``post_norm`` and ``next_norm`` are
    :class:`NormSpec`.  ``gate``: one value for each element (the shape of x), for each token (``[..., 1]``) or for each
    channel of a sample (``[B, 1, .., C]``, ``[1, .., C]`` or ``[C]``), through ``gate_activation`` (``"identity"``,
    ``"sigmoid"``, ``"tanh"``).  ``scale``: a vector of C values or a number.  ``p``, ``rng``: as for :func:`dropout`.
    Parameters (norm weights and biases, a scale vector) are of x's dtype or fp32.  ``y`` is the norm of ``out``
    before its rounding to x's dtype.

    Returns ``(out, y)``.  Differentiable in x, h, the gate and the parameters; gradients of what is broadcast are
    summed in fp32 in a fixed order.
    """
    return _native.host().residual_norm(x, h, post_norm, gate, gate_activation, scale, next_norm, p, rng)


__all__ = ["MAX_DIM", "NormSpec", "dropout", "norm", "residual_norm"]
