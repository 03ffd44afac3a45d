"""Host-side checks of the feed-forward operators, without a GPU: malformed calls are refused with a message before
anything touches a device, and the sizes that callers allocate by follow their definition."""
import ctypes
import struct

import pytest
import torch

#: p3d_residual and p3d_fp8_linear of include/pack3d_b200.h
RESIDUAL = struct.Struct("@2q9P2Q7iI3f4x")
LINEAR = struct.Struct("@3q3Pq5i4x")
DUMMY = 256   # a non-null, aligned stand-in: never dereferenced on these paths


def residual(rows=4, per_sample=0, x=DUMMY, h=DUMMY, gate=0, pw=0, pb=0, scale=0, nw=0, nb=0, dim=64, dtype=2, param=2,
             post=1, nxt=1, mode=0, act=0, threshold=0, post_eps=0.0, next_eps=0.0):
    return RESIDUAL.pack(rows, per_sample, x, h, gate, pw, pb, scale, nw, nb, 0, 0, 0, dim, dtype, param, post, nxt, mode,
                         act, threshold, post_eps, next_eps, 1.0)


@pytest.fixture(scope="module")
def lib():
    from pack3d_b200 import _native
    return _native.lib()


@pytest.mark.parametrize("change,text", [
    ({"dtype": 7}, b"dtype"), ({"param": 1}, b"parameters"), ({"rows": -1}, b"row count"), ({"dim": 0}, b"dim"),
    ({"post": 3}, b"norm"), ({"mode": 1}, b"gate"), ({"gate": DUMMY}, b"gate"), ({"act": 9}, b"gate"),
    ({"threshold": 65537}, b"threshold"), ({"post_eps": -1.0}, b"eps"), ({"h": 0}, b"needs h"),
    ({"h": 0, "post": 0, "nxt": 0}, b"nothing"), ({"mode": 2, "gate": DUMMY, "per_sample": 3}, b"samples")])
def test_residual_arguments(lib, change, text):
    assert lib.p3d_residual_fwd(residual(**change), DUMMY, DUMMY, 0, None) == 1
    assert text in lib.p3d_last_error()
    assert lib.p3d_residual_bwd_workspace(residual(**change)) == 0


def test_residual_limits_and_pointers(lib):
    assert lib.p3d_residual_fwd(residual(dim=16385), DUMMY, DUMMY, 0, None) == 2
    assert lib.p3d_residual_fwd(residual(rows=2 ** 31), DUMMY, DUMMY, 0, None) == 2
    assert lib.p3d_residual_fwd(residual(x=0), DUMMY, DUMMY, 0, None) == 1 and b"null" in lib.p3d_last_error()
    assert lib.p3d_residual_fwd(residual(), 0, DUMMY, 0, None) == 1
    assert lib.p3d_residual_fwd(residual(rows=0, x=0), 0, 0, 0, None) == 0      # nothing to do
    assert lib.p3d_residual_fwd(None, 0, 0, 0, None) == 1
    assert lib.p3d_residual_bwd(residual(), DUMMY, DUMMY, None, *[None] * 8, DUMMY, 1 << 30, None) == 1
    assert lib.p3d_residual_bwd(residual(nxt=0), DUMMY, DUMMY, DUMMY, *[None] * 8, DUMMY, 1 << 30, None) == 1
    assert b"next norm" in lib.p3d_last_error()


def test_row_limit_leaves_room_for_a_step(lib):
    """Row numbers are 32-bit in the kernels and go up to one step (under 1024 rows) past the last row."""
    assert lib.p3d_residual_fwd(residual(rows=2 ** 31 - 1), DUMMY, DUMMY, 0, None) == 2
    assert lib.p3d_residual_bwd_workspace(residual(rows=2 ** 31 - 1)) == 0


def test_dropout_arguments(lib):
    assert lib.p3d_dropout(DUMMY, DUMMY, 5, 4, 64, 0, None, 0, 0, None) == 1
    assert lib.p3d_dropout(DUMMY, DUMMY, 2, -1, 64, 0, None, 0, 0, None) == 1
    assert lib.p3d_dropout(DUMMY, DUMMY, 2, 2 ** 40, 2 ** 40, 0, None, 0, 0, None) == 1
    assert lib.p3d_dropout(DUMMY, DUMMY, 2, 4, 64, 70000, None, 0, 0, None) == 1
    assert lib.p3d_dropout(None, DUMMY, 2, 4, 64, 0, None, 0, 0, None) == 1
    assert lib.p3d_dropout(None, None, 2, 0, 64, 0, None, 0, 0, None) == 0


def test_fp8_sizes(lib):
    """512 scale bytes for every 128 rows and four blocks of 128 columns."""
    for rows, cols, want in ((1, 1, 512), (128, 512, 512), (129, 513, 4 * 512), (0, 5, 0), (300, 1100, 3 * 3 * 512)):
        assert lib.p3d_fp8_scale_bytes(rows, cols) == want
    assert lib.p3d_fp8_quantize_workspace(129, 100) == 2 * 100 * 4


def test_fp8_arguments(lib):
    quantize = lambda **k: lib.p3d_fp8_quantize(*[dict(x=DUMMY, dtype=2, rows=4, cols=64, square=0, q=DUMMY, pitch=64,  # noqa: E731
                                                       scales=DUMMY, qt=None, tp=0, ts=None, sums=None, st=0, ws=None, wb=0,
                                                       stream=None, **{}) | k][0].values())
    assert quantize(dtype=4) == 1 and quantize(rows=0) == 1 and quantize(x=None) == 1
    assert quantize(pitch=40) == 1 and b"pitch" in lib.p3d_last_error()
    assert quantize(pitch=72) == 1 and quantize(scales=None) == 1
    assert quantize(qt=DUMMY, ts=DUMMY, tp=2) == 1 and b"transposed" in lib.p3d_last_error()
    assert quantize(sums=DUMMY) == 4
    assert quantize(rows=65536 * 128) == 2
    args = (DUMMY, 64, DUMMY, DUMMY, 64, DUMMY, 4, 32, 64, None, 0, DUMMY, 2, None, 0, None)
    matmul = lambda at, v: lib.p3d_fp8_matmul(*(v if i == at else a for i, a in enumerate(args)))  # noqa: E731
    assert matmul(0, None) == 1 and matmul(6, 0) == 1 and matmul(1, 63) == 1 and matmul(4, 72) == 1
    assert matmul(12, 9) == 1 and matmul(0, 8) == 1 and b"aligned" in lib.p3d_last_error()
    assert matmul(6, 2 ** 40) == 2
    linear = LINEAR.pack(4, 64, 32, 0, 0, 0, 0, 2, 2, 2, 0, 0)
    assert lib.p3d_fp8_linear_fwd(linear, DUMMY, None, DUMMY, None, DUMMY, 1 << 30, None) == 1
    assert lib.p3d_fp8_linear_fwd(LINEAR.pack(0, 64, 32, DUMMY, 0, 0, 0, 2, 2, 2, 0, 0), DUMMY, None, DUMMY, None, DUMMY,
                                  1 << 30, None) == 1
    assert lib.p3d_fp8_linear_bwd(linear, DUMMY, None, DUMMY, None, None, DUMMY, 1 << 30, None) == 1


def test_struct_layouts_match_the_header(tmp_path):
    import subprocess
    from pathlib import Path
    header = Path(__file__).resolve().parents[1] / "include" / "pack3d_b200.h"
    probe = ('#include <stddef.h>\n#include <stdio.h>\n#include "%s"\nint main(void){printf("%%zu %%zu %%zu %%zu %%zu\\n",'
             'sizeof(p3d_residual),offsetof(p3d_residual,dim),offsetof(p3d_residual,scale_value),'
             'sizeof(p3d_fp8_linear),offsetof(p3d_fp8_linear,dtype));}' % header)
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-x", "c", "-", "-o", str(exe)], input=probe, text=True, check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [RESIDUAL.size, 104, 144, LINEAR.size, 56]


def test_cpu_tensors_are_refused_not_computed():
    from pack3d_b200 import NormSpec, dropout, fp8_linear, norm, quantize, quantize_weight, residual_norm
    x = torch.randn(4, 64)
    for call in (lambda: dropout(x, 0.5, (1, 2)), lambda: norm(x, NormSpec()), lambda: residual_norm(x, x),
                 lambda: fp8_linear(x, x), lambda: quantize(x), lambda: quantize_weight(x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_host_module_is_built_beside_the_library():
    from pack3d_b200 import _native
    module = _native.host()
    assert {"dropout", "norm", "residual_norm", "fp8_linear"} <= set(dir(module))
    with pytest.raises(ValueError, match="tensor"):
        module.dropout(3, 0.5, (1, 2))
    with pytest.raises(ValueError, match="takes"):
        module.norm(torch.zeros(2))
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_tangents_are_refused():
    """A forward-mode derivative is refused before anything else, not dropped."""
    import torch.autograd.forward_ad as forward_ad
    from pack3d_b200 import NormSpec, dropout, fp8_linear, norm, residual_norm
    x = torch.randn(4, 64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: dropout(dual, 0.5, (1, 2)), lambda: norm(dual, NormSpec()), lambda: residual_norm(dual, x),
                     lambda: residual_norm(x, dual), lambda: fp8_linear(dual, x), lambda: fp8_linear(x, dual),
                     lambda: fp8_linear(x, x, dual[0])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_fp8_matrix_refuses_parts_that_do_not_fit():
    """Kernels take addresses and extents from it: values, scales, rows and columns have to belong together."""
    from pack3d_b200 import Fp8Matrix
    values, scales = torch.zeros(130, 80, dtype=torch.float8_e4m3fn), torch.zeros(1024, dtype=torch.uint8)
    assert Fp8Matrix(values, scales, 130, 70).shape == (130, 70)
    for bad in (values.view(torch.uint8), values[:, :64], values[:129], values[0], values.t().contiguous(), None,
                torch.zeros(130, 72, dtype=torch.float8_e4m3fn), torch.zeros(130, 64, dtype=torch.float8_e4m3fn)):
        with pytest.raises(ValueError, match="values of a 130 x 70"):
            Fp8Matrix(bad, scales, 130, 70)
    for bad in (scales[:512], torch.zeros(2048, dtype=torch.uint8)[::2], scales.view(torch.int8), None, scales.to("meta")):
        with pytest.raises(ValueError, match="scales of a 130 x 70"):
            Fp8Matrix(values, bad, 130, 70)
    for rows, cols in ((128, 70), (131, 70), (130, 0), (130, 81), (0, 70)):
        with pytest.raises(ValueError):
            Fp8Matrix(values, scales, rows, cols)


def test_scale_bytes_agree_with_the_library(lib):
    from pack3d_b200.fp8 import _scale_bytes
    for rows, cols in ((1, 1), (128, 512), (129, 513), (300, 1100), (4096, 16384)):
        assert _scale_bytes(rows, cols) == lib.p3d_fp8_scale_bytes(rows, cols)


def test_matmul_bias_that_wants_a_gradient_is_refused():
    import torch.autograd.forward_ad as forward_ad
    from pack3d_b200.fp8 import _check_bias
    bias = torch.zeros(3, requires_grad=True)
    with pytest.raises(ValueError, match="no gradients"):
        _check_bias(bias, 3, bias.device)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="no gradients"):
        _check_bias(forward_ad.make_dual(bias.detach(), torch.ones(3)), 3, bias.device)
    with torch.no_grad():
        assert _check_bias(bias, 3, bias.device).shape == (3,)


@pytest.mark.parametrize("extents", [(2 ** 62, 64, 32), (64, 2 ** 62, 32), (64, 32, 2 ** 62), (2 ** 40, 2 ** 40, 2 ** 40),
                                     (2 ** 30 + 1, 64, 32)])
def test_linear_extents_whose_sizes_would_overflow(lib, extents):
    args = LINEAR.pack(*extents, DUMMY, 0, 0, 0, 2, 2, 2, 1, 1)
    for size in (lib.p3d_fp8_linear_saved, lib.p3d_fp8_linear_fwd_workspace, lib.p3d_fp8_linear_bwd_workspace):
        assert size(args) == 0
    assert lib.p3d_fp8_linear_fwd(args, DUMMY, None, DUMMY, DUMMY, DUMMY, 1 << 40, None) == 2
    assert lib.p3d_fp8_linear_bwd(args, DUMMY, DUMMY, DUMMY, DUMMY, None, DUMMY, 1 << 40, None) == 2
    assert b"too large" in lib.p3d_last_error()
