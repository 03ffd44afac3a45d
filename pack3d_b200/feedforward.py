"""The feed-forward half of a transformer block behind :class:`~pack3d_b200.PACK3DAttention`, on its residual stream.

:class:`FeedForward` runs :func:`~pack3d_b200.norm`, :func:`~pack3d_b200.fp8_linear`, :func:`~pack3d_b200.residual_norm` and
its dropout together.  No counterpart in the reference, whose package ends at the attention layer
(``src/pack3d/attention.py:89``).
"""
import math

import torch
from torch import nn

from .fp8 import fp8_linear, quantize_weight
from .residual import NormSpec, norm, residual_norm


class FeedForward(nn.Module):
    """``x + residual_scale * dropout(post_norm(W2 gelu(W1 pre_norm(x) + b1) + b2) * act(gate))``.

    Input / output ``[..., dim]`` on a CUDA sm_100 device.  Both products are 8-bit blocks with power-of-two scales, in
    training with both gradients; norms, gate, dropout, scale and residual are one kernel a direction.

    A stack of blocks hands the norm on: ``forward(x, normed=y, next_norm=spec)`` takes the ``pre_norm`` of x that the
    block before made and returns ``(out, next_norm(out))`` from one kernel::

        y = None
        for i, layer in enumerate(layers):
            following = layers[i + 1].pre_norm if i + 1 < len(layers) else None
            x, y = layer(x, normed=y, next_norm=following, rng=(seed, step * len(layers) + i))

    For serving, :meth:`keep_8bit` quantises the weights once; :meth:`forward` then runs without gradients and without
    dropout from those (a single token included), in ``train()`` too, until :meth:`keep_8bit` is called again with
    ``keep=False``.
    """

    def __init__(self, dim, hidden, *, norm="layer", eps=1e-6, dropout=0.0, residual_scale=0.1,
                 gate_activation="identity"):
        super().__init__()
        if any(type(v) is not int or v <= 0 for v in (dim, hidden)):
            raise ValueError("dimensions must be positive integers")
        if norm not in ("layer", "rms"):
            raise ValueError("norm must be layer or rms")
        if not 0.0 <= dropout < 1.0:
            raise ValueError("dropout must lie in [0, 1)")
        if not math.isfinite(residual_scale):
            raise ValueError("residual_scale must be finite")
        self.dim, self.hidden, self.kind, self.eps = dim, hidden, norm, float(eps)
        self.dropout, self.gate_activation = float(dropout), gate_activation
        self.pre_weight = nn.Parameter(torch.ones(dim))
        self.post_weight = nn.Parameter(torch.ones(dim))
        self.pre_bias = nn.Parameter(torch.zeros(dim)) if norm == "layer" else None
        self.post_bias = nn.Parameter(torch.zeros(dim)) if norm == "layer" else None
        self.scale = nn.Parameter(torch.full((dim,), float(residual_scale)))
        self.w1 = nn.Parameter(torch.empty(hidden, dim))
        self.b1 = nn.Parameter(torch.zeros(hidden))
        self.w2 = nn.Parameter(torch.empty(dim, hidden))
        self.b2 = nn.Parameter(torch.zeros(dim))
        for w in (self.w1, self.w2):
            nn.init.normal_(w, std=1 / math.sqrt(w.shape[1]))
        self._kept = None
        self._kept_from = None

    @property
    def pre_norm(self):
        """The norm before the block, for the ``next_norm`` of the block before it."""
        return NormSpec(self.pre_weight, self.pre_bias, self.kind, self.eps)

    @property
    def post_norm(self):
        return NormSpec(self.post_weight, self.post_bias, self.kind, self.eps)

    def keep_8bit(self, keep=True):
        """Quantise both weights now and serve from them (``keep=False``: go back to the parameters); returns self.

        Weights that change afterwards (``load_state_dict``, in-place updates, ``.to()``, another parameter in their place)
        are quantised again by the next :meth:`forward`, into the same memory, which captured graphs read.  PyTorch counts
        neither writes through ``.data`` nor the steps of fused optimizers: after those, call this again.  A weight that is
        taken out (None, or of another shape) leaves what was kept of it.
        """
        weights = (self.w1, self.w2)
        self._kept = tuple(quantize_weight(w) for w in weights) if keep else None
        self._kept_from = [(w, w._version) for w in weights] if keep else None
        return self

    def _apply(self, fn, recurse=True):   # .to(), .half(), ..: other values under the same parameters
        result = super()._apply(fn, recurse)
        if self._kept is not None:
            self._kept_from = [(None, 0)] * 2
        return result

    def _serving(self):
        """The kept weights, brought up to date with the parameters."""
        weights = (self.w1, self.w2)
        for i, (w, (seen, version)) in enumerate(zip(weights, self._kept_from)):
            if w is seen and (w is None or w._version == version):
                continue
            if w is not None and w.is_cuda and w.shape == self._kept[i].shape:
                if torch.cuda.is_current_stream_capturing():
                    raise ValueError("weights kept in 8 bits have changed: call keep_8bit() before the capture")
                new, old = quantize_weight(w), self._kept[i]
                if old.device == new.device:
                    old.values.view(torch.uint8).copy_(new.values.view(torch.uint8))
                    old.scales.copy_(new.scales)
                else:
                    self._kept = (*self._kept[:i], new, *self._kept[i + 1:])
            self._kept_from[i] = (w, 0 if w is None else w._version)
        return self._kept

    def forward(self, x, *, normed=None, gate=None, next_norm=None, rng=None):
        """``(out, next_norm(out))``, the second None without ``next_norm``.  ``gate`` as for :func:`residual_norm`;
        ``rng = (seed, offset)`` is needed where the module drops out in training, a new one for every call."""
        p = self.dropout if self.training and self._kept is None else 0.0
        if p and rng is None:
            raise ValueError("dropout in training needs rng=(seed, offset)")
        if self._kept is not None and torch.is_grad_enabled():
            raise ValueError("weights kept in 8 bits have no gradients: call under torch.no_grad()")
        w1, w2 = self._serving() if self._kept is not None else (self.w1, self.w2)
        y = norm(x, self.pre_norm) if normed is None else normed
        h = torch.nn.functional.gelu(fp8_linear(y, w1, self.b1))
        h = fp8_linear(h, w2, self.b2)
        return residual_norm(x, h, post_norm=self.post_norm, gate=gate, gate_activation=self.gate_activation,
                             scale=self.scale, next_norm=next_norm, p=p, rng=rng)
