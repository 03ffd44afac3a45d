"""Linear layers in 8-bit floating point with one power-of-two scale for each block of 128.

* :class:`Fp8Matrix` -- e4m3 values and their scales as the tensor cores read them.
* :func:`quantize` / :func:`quantize_weight` -- blocks of 1 x 128 (activations) and 128 x 128 (weights).
* :func:`fp8_matmul` -- ``a b^T`` of two such matrices, fp32 accumulation, one rounding at the end.
* :func:`fp8_linear` -- ``x W^T + bias`` for training (both gradients in the same products) or from a kept weight.

No counterpart in the reference, whose projections are 16- or 32-bit (``attention.py:37-51``).  A block's scale is the
smallest power of two that brings its largest finite magnitude to at most 448, so scaling is exact and e4m3's rounding
to nearest even is the only one; products are exact in fp32.  NaN and infinities become NaN and set no scale.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _native
from ._validation import check_cuda

BLOCK = 128


def _scale_bytes(rows, cols):
    """512 for every 128 rows and every four blocks of columns."""
    return -(-rows // BLOCK) * -(-cols // (4 * BLOCK)) * 512


class Fp8Matrix:
    """``values`` [rows, pitch] (``torch.float8_e4m3fn``, contiguous, pitch a multiple of 16, columns from ``cols`` on
    unused) and ``scales`` (contiguous bytes e + 127 of 2^e, one for each row and block of 128 columns, in the order of
    ``p3d_fp8_quantize``), on one device."""

    __slots__ = ("values", "scales", "rows", "cols")

    def __init__(self, values, scales, rows, cols):
        self.values, self.scales, self.rows, self.cols = values, scales, int(rows), int(cols)
        self._check()

    def _check(self):
        """The kernels take addresses, rows and columns from here: refuse what does not fit together."""
        v, s = self.values, self.scales
        if not (isinstance(v, torch.Tensor) and v.dtype == torch.float8_e4m3fn and v.ndim == 2 and v.is_contiguous()
                and v.shape[0] == self.rows >= 1 and v.shape[1] >= self.cols >= 1 and v.shape[1] % 16 == 0):
            raise ValueError(f"values of a {self.rows} x {self.cols} Fp8Matrix must be contiguous float8_e4m3fn [rows, pitch], "
                             "the pitch a multiple of 16 and at least the columns")
        if not (isinstance(s, torch.Tensor) and s.dtype == torch.uint8 and s.is_contiguous() and s.device == v.device
                and s.numel() == _scale_bytes(self.rows, self.cols)):
            raise ValueError(f"scales of a {self.rows} x {self.cols} Fp8Matrix must be {_scale_bytes(self.rows, self.cols)} "
                             "contiguous uint8 on the device of its values")

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    @property
    def device(self):
        return self.values.device

    def exponents(self):
        """int32 [rows, ceil(cols / 128)]: the e of each block's scale 2^e."""
        blocks = -(-self.cols // BLOCK)
        tiles, groups = -(-self.rows // BLOCK), -(-blocks // 4)
        t = self.scales.view(tiles, groups, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles * BLOCK, groups * 4)
        return t[:self.rows, :blocks].to(torch.int32) - 127

    def dequantize(self, dtype=torch.float32):
        """The values that the bytes stand for, [rows, cols], rounded to ``dtype`` (infinite where it cannot hold
        them: a block's largest value may round up past fp32's range)."""
        scale = ((self.exponents() + 127) << 23).view(torch.float32).to(torch.float64)   # 2^e from its bits
        scale = scale.repeat_interleave(BLOCK, 1)[:, :self.cols]
        return (self.values[:, :self.cols].to(torch.float64) * scale).to(dtype)

    @staticmethod
    def _empty(rows, cols, device):
        pitch = -(-cols // 16) * 16
        return Fp8Matrix(torch.empty((rows, pitch), dtype=torch.float8_e4m3fn, device=device),
                         torch.empty(_scale_bytes(rows, cols), dtype=torch.uint8, device=device),
                         rows, cols)


def _check_matrix(x, what):
    check_cuda(x)
    if x.ndim != 2 or x.shape[0] < 1 or x.shape[1] < 1:
        raise ValueError(f"{what} needs a matrix with at least one row and one column, got {list(x.shape)}")


def _quantize(x, square=False, rows=True, transposed=False, sums=None):
    """(q or None, qt or None) of a contiguous matrix; `sums`: a vector for the sums over its rows."""
    m, n = x.shape
    q = Fp8Matrix._empty(m, n, x.device) if rows else None
    qt = Fp8Matrix._empty(n, m, x.device) if transposed else None
    lib = _native.lib()
    with _native.on(x.device) as stream:
        ws = None
        if sums is not None:
            ws = torch.empty(max(16, lib.p3d_fp8_quantize_workspace(m, n)), dtype=torch.uint8, device=x.device)
        _native.check(lib.p3d_fp8_quantize(
            x.data_ptr(), _native.DTYPE_CODE[x.dtype], m, n, 1 if square else 0,
            q.values.data_ptr() if q else None, q.values.shape[1] if q else 0, q.scales.data_ptr() if q else None,
            qt.values.data_ptr() if qt else None, qt.values.shape[1] if qt else 0, qt.scales.data_ptr() if qt else None,
            None if sums is None else sums.data_ptr(), 0 if sums is None else _native.DTYPE_CODE[sums.dtype],
            None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), stream), "p3d_fp8_quantize")
    return q, qt


def quantize(x):
    """:class:`Fp8Matrix` of a matrix with one scale for each row and block of 128 columns."""
    _check_matrix(x, "quantize")
    return _quantize(x.detach().contiguous())[0]


def quantize_weight(weight):
    """:class:`Fp8Matrix` of a weight [out, in] with one scale for each 128 x 128 block (repeated for its rows), as
    :func:`fp8_linear` quantises it: keep it to serve from 8-bit weights."""
    _check_matrix(weight, "quantize_weight")
    return _quantize(weight.detach().contiguous(), square=True)[0]


def _matmul(a, b, bias, dtype):
    out = torch.empty((a.rows, b.rows), dtype=dtype, device=a.device)
    lib = _native.lib()
    with _native.on(a.device) as stream:
        need = lib.p3d_fp8_matmul_workspace(a.rows, b.rows, a.cols)
        ws = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None
        _native.check(lib.p3d_fp8_matmul(
            a.values.data_ptr(), a.values.shape[1], a.scales.data_ptr(), b.values.data_ptr(), b.values.shape[1],
            b.scales.data_ptr(), a.rows, b.rows, a.cols, None if bias is None else bias.data_ptr(),
            0 if bias is None else _native.DTYPE_CODE[bias.dtype], out.data_ptr(), _native.DTYPE_CODE[dtype],
            None if ws is None else ws.data_ptr(), need, stream), "p3d_fp8_matmul")
    return out


def _check_bias(bias, n, device):
    if bias is None:
        return None
    if bias.shape != (n,) or bias.device != device or bias.dtype not in _native.DTYPE_CODE:
        raise ValueError(f"bias must be {n} fp32, fp16 or bf16 values on the input's device")
    if bias.requires_grad and torch.is_grad_enabled() or forward_ad.unpack_dual(bias).tangent is not None:
        raise ValueError("fp8_matmul has no gradients: pass bias.detach(), or call under torch.no_grad()")
    return bias.contiguous()


def fp8_matmul(a, b, *, bias=None, dtype=torch.bfloat16):
    """``a b^T`` (``+ bias``) as [a.rows, b.rows] of ``dtype`` (fp32, fp16, bf16) for two :class:`Fp8Matrix` of the same
    number of columns.  Products and sums in fp32; the order of the sum depends on the extents alone.  No gradients: a
    bias that wants one is refused."""
    if not (isinstance(a, Fp8Matrix) and isinstance(b, Fp8Matrix)):
        raise ValueError("fp8_matmul takes two Fp8Matrix")
    a._check()   # the attributes may have been set since
    b._check()
    if a.cols != b.cols or a.device != b.device:
        raise ValueError(f"operands must have the same columns and device, got {list(a.shape)} and {list(b.shape)}")
    if dtype not in _native.DTYPE_CODE:
        raise ValueError("dtype must be fp32, fp16 or bf16")
    return _matmul(a, b, _check_bias(bias, b.rows, a.device), dtype)


def fp8_linear(x, weight, bias=None):
    """``x weight^T + bias`` over the last dimension of ``x`` with both operands in 8-bit blocks.

    ``x`` [..., in] fp32, fp16 or bf16.  ``weight`` [out, in] is a tensor, quantised in the call (training: its gradient
    and x's are products of 8-bit blocks too), or an :class:`Fp8Matrix` from :func:`quantize_weight` (serving; no
    gradients).  Blocks: x and dy 1 x 128 along the dimension that is summed over (for the weight's gradient that
    is the tokens), the weight 128 x 128.  The result has x's dtype, gradients their inputs'; the bias's gradient is
    summed in fp32.  Differentiable once, in reverse mode; second and forward-mode derivatives are refused.
    """
    if isinstance(weight, Fp8Matrix):
        return _native.host().fp8_linear(x, None, bias, weight.values, weight.scales, weight.rows, weight.cols)
    return _native.host().fp8_linear(x, weight, bias, None, None, 0, 0)


__all__ = ["BLOCK", "Fp8Matrix", "fp8_linear", "fp8_matmul", "quantize", "quantize_weight"]
