"""The parts of a transformer block around its matrix products: norms before and after the block with its gate,
dropout, residual scale and residual, and dropout by itself, each one kernel in each direction.

* :func:`norm` -- RMS or layer norm over the last dimension.
* :func:`residual_norm` -- ``out = x + scale * dropout(post_norm(h) * act(gate))`` and ``y = next_norm(out)``.
* :func:`dropout` -- counter-based: the mask is a function of (seed, offset) and the element's place, made again in the
  backward pass and never stored.

No counterpart in the reference, whose layer ends at its own residual (``attention.py:89``).  fp32, fp16 and bf16 CUDA
tensors, any leading shape, up to 16,384 columns; statistics, sums and gradients of parameters in fp32, each value
rounded once where it is stored.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native
from ._validation import check_cuda

MAX_DIM = 16384
_KINDS = {"rms": 1, "layer": 2}
_ACTIVATIONS = {"identity": 0, "sigmoid": 1, "tanh": 2}
_GATE_ELEMENT, _GATE_SAMPLE, _GATE_TOKEN = 1, 2, 3


class NormSpec(NamedTuple):
    """A norm over the last dimension: ``kind`` ``"rms"`` (``z / sqrt(mean(z^2) + eps)``) or ``"layer"``
    (``(z - mean) / sqrt(var + eps)``), times ``weight`` plus ``bias`` (either may be None)."""
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    kind: str = "rms"
    eps: float = 1e-6


# ------------------------------------------------------------------------------- arguments
def _check_input(x, what):
    if x.ndim < 1:
        raise ValueError(f"{what} needs at least one dimension")
    check_cuda(x)
    if not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError(f"{what}: the last dimension must be 1 to {MAX_DIM}, got {x.shape[-1]}")


def _check_spec(spec, x, what):
    if not isinstance(spec, NormSpec):
        raise ValueError(f"{what} must be a NormSpec")
    if spec.kind not in _KINDS:
        raise ValueError(f"{what}: kind must be 'rms' or 'layer'")
    if not (math.isfinite(spec.eps) and spec.eps >= 0):
        raise ValueError(f"{what}: eps must be finite and not negative")
    _check_vector(spec.weight, x, what)
    _check_vector(spec.bias, x, what)


def _check_vector(t, x, what):
    if t is None:
        return
    if t.shape != x.shape[-1:]:
        raise ValueError(f"{what}: parameters must have shape [{x.shape[-1]}], got {list(t.shape)}")
    if t.device != x.device:
        raise ValueError(f"{what}: parameters and input must be on the same device")
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise ValueError(f"{what}: parameters must be {x.dtype} or torch.float32, got {t.dtype}")


def _threshold(p):
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout probability must lie between 0 and 1")
    return round(65536 * p)


def _rng(rng, device):
    """``(tensor or None, seed, offset)`` of a ``(seed, offset)`` pair or an int64 CUDA tensor of two."""
    if isinstance(rng, torch.Tensor):
        if rng.dtype != torch.int64 or rng.numel() != 2 or rng.device != device or not rng.is_contiguous():
            raise ValueError("rng must hold (seed, offset): two contiguous int64 on the input's device")
        return rng, 0, 0
    if rng is None:
        raise ValueError("dropout needs rng: (seed, offset) or an int64 tensor of the two")
    try:
        seed, offset = (int(v) for v in rng)
    except (TypeError, ValueError):
        raise ValueError("rng must be (seed, offset) or an int64 tensor of the two") from None
    return None, seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF


def _address(t):
    return 0 if t is None else t.data_ptr()


# ------------------------------------------------------------------------------- dropout
def _run_dropout(x, threshold, rng, seed, offset):
    x = x.contiguous()
    y = torch.empty_like(x)
    dim = x.shape[-1] if x.ndim else 1
    rows = x.numel() // dim if dim else 0
    with _native.on(x.device) as stream:
        status = _native.lib().p3d_dropout(x.data_ptr(), y.data_ptr(), _native.DTYPE_CODE[x.dtype], rows, dim, threshold,
                                           _address(rng) or None, seed, offset, stream)
    if status:
        _native.check(status, "p3d_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, threshold, rng, seed, offset):
        ctx.save_for_backward(rng)
        ctx.meta = (threshold, seed, offset)
        return _run_dropout(x, threshold, rng, seed, offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        threshold, seed, offset = ctx.meta
        return _run_dropout(dy, threshold, ctx.saved_tensors[0], seed, offset), None, None, None, None


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
    check_cuda(x)
    threshold = _threshold(p)
    tensor, seed, offset = _rng(rng, x.device)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dropout.apply(x, threshold, tensor, seed, offset)
    return _run_dropout(x, threshold, tensor, seed, offset)


# ------------------------------------------------------------------------------- norms and residual
class _Plan(NamedTuple):
    """What a call is, apart from its tensors."""
    post: int
    post_eps: float
    next: int
    next_eps: float
    gate_mode: int
    gate_act: int
    rows_per_sample: int
    scale_value: float
    threshold: int
    seed: int
    offset: int


def _pack(plan, x, h, gate, post_w, post_b, scale, next_w, next_b, rng):
    dim = x.shape[-1]
    code = _native.DTYPE_CODE[x.dtype]
    param = next((t for t in (post_w, post_b, scale, next_w, next_b) if t is not None), x)
    return _native.RESIDUAL.pack(
        x.numel() // dim, plan.rows_per_sample, x.data_ptr(), _address(h), _address(gate), _address(post_w),
        _address(post_b), _address(scale), _address(next_w), _address(next_b), _address(rng), plan.seed, plan.offset,
        dim, code, _native.DTYPE_CODE[param.dtype], plan.post, plan.next, plan.gate_mode, plan.gate_act,
        plan.threshold, plan.post_eps, plan.next_eps, plan.scale_value)


def _run_forward(plan, tensors, save):
    x, h = tensors[0], tensors[1]
    out = None if h is None else torch.empty_like(x)
    y = torch.empty_like(x) if plan.next else None
    stats = x.new_empty((x.numel() // x.shape[-1], 4), dtype=torch.float32) if save else None
    if x.numel() == 0:
        return out, y, stats
    with _native.on(x.device) as stream:
        status = _native.lib().p3d_residual_fwd(_pack(plan, *tensors), _address(out), _address(y), _address(stats),
                                                stream)
    if status:
        _native.check(status, "p3d_residual_fwd")
    return out, y, stats


class _Residual(torch.autograd.Function):
    """inputs: plan, rng, x, h, gate, post_w, post_b, scale, next_w, next_b (h None: only the next norm)."""

    @staticmethod
    def forward(ctx, plan, rng, *tensors):
        ctx.set_materialize_grads(False)
        out, y, stats = _run_forward(plan, (*tensors, rng), True)
        ctx.plan = plan
        ctx.save_for_backward(rng, stats, *tensors)
        return out, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dy):
        rng, stats, *tensors = ctx.saved_tensors
        plan, x, h, gate = ctx.plan, tensors[0], tensors[1], tensors[2]
        need = ctx.needs_input_grad[2:]
        if dout is None and dy is None:
            return (None,) * 10
        if x.numel() == 0:
            return None, None, *(torch.zeros_like(t) if n else None for t, n in zip(tensors, need))
        dout, dy = (None if g is None else g.contiguous() for g in (dout, dy))
        # x, h, gate, scale, post weight and bias, next weight and bias
        grads = [torch.empty_like(t) if n else None for t, n in zip(tensors, need)]
        packed = _pack(plan, *tensors, rng)
        lib = _native.lib()
        with _native.on(x.device) as stream:
            need = lib.p3d_residual_bwd_workspace(packed)
            ws = stats.new_empty(need // 4)
            dx, dh, dgate, dpw, dpb, dscale, dnw, dnb = map(_address, grads)
            status = lib.p3d_residual_bwd(packed, _address(dout), _address(dy), stats.data_ptr(), dx, dh, dgate, dscale,
                                          dpw, dpb, dnw, dnb, ws.data_ptr(), need, stream)
        if status:
            _native.check(status, "p3d_residual_bwd")
        return None, None, *grads


def _call(plan, rng, tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return _Residual.apply(plan, rng, *tensors)
    return _run_forward(plan, (*tensors, rng), False)[:2]


def _same_params(*params):
    """The parameters contiguous and of one dtype: where they differ, all in fp32."""
    dtype = None
    for t in params:
        if t is not None:
            if dtype is not None and t.dtype != dtype:
                params = [None if t is None else t.float() for t in params]
                break
            dtype = t.dtype
    return [t if t is None or t.is_contiguous() else t.contiguous() for t in params]


def norm(x, spec):
    """``spec`` (:class:`NormSpec`) of ``x`` over its last dimension, differentiable in ``x``, weight and bias."""
    _check_input(x, "norm")
    _check_spec(spec, x, "norm")
    w, b = _same_params(spec.weight, spec.bias)
    plan = _Plan(0, 0.0, _KINDS[spec.kind], float(spec.eps), 0, 0, 0, 1.0, 0, 0, 0)
    return _call(plan, None, (x.contiguous(), None, None, None, None, None, w, b))[1]


def _gate_mode(gate, x):
    """(mode, rows of one sample, the gate as the kernel takes it)."""
    if gate.device != x.device or gate.dtype != x.dtype:
        raise ValueError("gate must have the dtype and device of x")
    rows = x.numel() // x.shape[-1]
    if gate.shape == x.shape:
        return _GATE_ELEMENT, 0, gate.contiguous()
    if gate.shape == (*x.shape[:-1], 1):
        return _GATE_TOKEN, 0, gate.contiguous()
    if gate.shape[-1:] == x.shape[-1:] and (gate.ndim == 1 or gate.ndim == x.ndim):
        lead = gate.shape[:-1]
        if all(n == 1 for n in lead):
            return _GATE_SAMPLE, max(rows, 1), gate.contiguous()
        if lead[0] == x.shape[0] and all(n == 1 for n in lead[1:]):
            return _GATE_SAMPLE, max(rows // x.shape[0], 1), gate.contiguous()
    raise ValueError(f"gate must have the shape of x {list(x.shape)}, one value for each token {[*x.shape[:-1], 1]}, "
                     f"or one vector for each sample or for all; got {list(gate.shape)}")


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
    _check_input(x, "residual_norm")
    if h.shape != x.shape or h.dtype != x.dtype or h.device != x.device:
        raise ValueError("h must have the shape, dtype and device of x")
    post = post_norm if post_norm is not None else NormSpec()
    nxt = next_norm if next_norm is not None else NormSpec()
    if post_norm is not None:
        _check_spec(post, x, "post_norm")
    if next_norm is not None:
        _check_spec(nxt, x, "next_norm")
    if gate_activation not in _ACTIVATIONS:
        raise ValueError("gate_activation must be 'identity', 'sigmoid' or 'tanh'")
    value = 1.0
    if isinstance(scale, torch.Tensor):
        _check_vector(scale, x, "scale")
    elif scale is not None:
        value, scale = float(scale), None
    mode, per_sample = 0, 0
    if gate is not None:
        mode, per_sample, gate = _gate_mode(gate, x)
    threshold = _threshold(p)
    tensor, seed, offset = _rng(rng, x.device) if threshold else (None, 0, 0)
    pw, pb, scale, nw, nb = _same_params(post.weight, post.bias, scale, nxt.weight, nxt.bias)
    plan = _Plan(_KINDS[post.kind] if post_norm is not None else 0, float(post.eps),
                 _KINDS[nxt.kind] if next_norm is not None else 0, float(nxt.eps), mode,
                 _ACTIVATIONS[gate_activation], per_sample, value, threshold, seed, offset)
    return _call(plan, tensor, (x.contiguous(), h.contiguous(), gate, pw, pb, scale, nw, nb))


__all__ = ["MAX_DIM", "NormSpec", "dropout", "norm", "residual_norm"]
