"""Host-side checks of attention over ordered sequences, without a GPU: malformed calls are refused with a message before
anything touches a device."""
import ctypes
import struct
import subprocess
from pathlib import Path

import pytest
import torch

#: p3d_norm_rotate, p3d_sequence and p3d_cache of include/pack3d_b200.h
ROTATE = struct.Struct("@2P2P2P2q2qP4qd2i2i2i2f4i3i4x")
SEQUENCE = struct.Struct("@3P2q2q2q2P2q6if4x")
CACHE = struct.Struct("@2P2PP2q6i")
DUMMY = 256   # a non-null, aligned stand-in: never dereferenced on these paths
PAIR = struct.Struct("@2q")


@pytest.fixture(scope="module")
def lib():
    from pack3d_b200 import _native
    return _native.lib()


def rotate(x0=DUMMY, x1=DUMMY, positions=DUMMY, tokens=4, rows=4, base=1e4, h0=2, h1=1, kind=(1, 1), pd=(2, 2), eps=(0.0, 0.0), dim=64,
           dtype=2, axes=1, pos=8, pairs=(32, 0, 0)):
    return ROTATE.pack(x0, x1, 0, 0, 0, 0, 128, 64, 64, 64, positions, 1, 1, tokens, rows, base, h0, h1, *kind, *pd, *eps, dim, dtype, axes,
                       pos, *pairs)


def sequence(q=DUMMY, k=DUMMY, v=DUMMY, stride=(128, 64), qo=DUMMY, ko=DUMMY, q_rows=4, k_rows=4, sequences=1, heads=2, kv=1, dim=64,
             dtype=2, causal=1, scale=0.1):
    return SEQUENCE.pack(q, k, v, *stride, *stride, *stride, qo, ko, q_rows, k_rows, sequences, heads, kv, dim, dtype, causal, scale)


def cache(k=DUMMY, v=DUMMY, ks=0, vs=0, table=DUMMY, pages=4, stride=2, width=2, sequences=1, heads=1, page=16, dim=64, dtype=2):
    return CACHE.pack(k, v, ks, vs, table, pages, stride, width, sequences, heads, page, dim, dtype)


def test_struct_layouts_match_the_header(tmp_path):
    header = Path(__file__).resolve().parents[1] / "include" / "pack3d_b200.h"
    probe = ('#include <stddef.h>\n#include <stdio.h>\n#include "%s"\nint main(void){printf("%%zu %%zu %%zu %%zu %%zu %%zu %%zu %%zu\\n",'
             'sizeof(p3d_norm_rotate),offsetof(p3d_norm_rotate,base),offsetof(p3d_norm_rotate,pairs),'
             'sizeof(p3d_sequence),offsetof(p3d_sequence,sequences),offsetof(p3d_sequence,scale),'
             'sizeof(p3d_cache),offsetof(p3d_cache,table_width));}' % header)
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-x", "c", "-", "-o", str(exe)], input=probe, text=True, check=True)
    out = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert out == [ROTATE.size, 120, 176, SEQUENCE.size, 104, 128, CACHE.size, 56]


@pytest.mark.parametrize("change,text", [
    ({"dtype": 5}, b"dtype"), ({"dim": 63}, b"even"), ({"dim": 258}, b"even"), ({"h0": 0}, b"heads"), ({"tokens": -1}, b"token"),
    ({"axes": 4}, b"axes"), ({"pos": 2}, b"int32"), ({"base": 0.5}, b"base"), ({"base": float("nan")}, b"base"), ({"pairs": (33, 0, 0)}, b"pairs"),
    ({"pairs": (-1, 0, 0)}, b"pairs"), ({"kind": (3, 1)}, b"norm"), ({"eps": (-1.0, 0.0)}, b"eps"), ({"pd": (1, 2)}, b"parameters"),
    ({"x0": 0}, b"null"), ({"positions": 0}, b"null"), ({"rows": 0}, b"token")])
def test_rotate_arguments(lib, change, text):
    assert lib.p3d_norm_rotate_fwd(rotate(**change), DUMMY, DUMMY, None) == 1
    assert text in lib.p3d_last_error()
    assert lib.p3d_norm_rotate_bwd_workspace(rotate(**change)) == 0


def test_rotate_limits(lib):
    assert lib.p3d_norm_rotate_fwd(None, DUMMY, DUMMY, None) == 1
    assert lib.p3d_norm_rotate_fwd(rotate(tokens=2 ** 31), DUMMY, DUMMY, None) == 2
    assert lib.p3d_norm_rotate_fwd(rotate(tokens=2 ** 30, rows=2 ** 30), DUMMY, DUMMY, None) == 2


@pytest.mark.parametrize("change,text", [
    ({"dtype": 0}, b"f16 or bf16"), ({"dim": 60}, b"multiple of 8"), ({"dim": 136}, b"multiple of 8"), ({"heads": 3, "kv": 2}, b"multiple"),
    ({"sequences": -1}, b"counts"), ({"q_rows": -1}, b"counts"), ({"scale": 0.0}, b"scale"), ({"scale": float("inf")}, b"scale"),
    ({"sequences": 0}, b"without a sequence"), ({"qo": 0}, b"offsets"), ({"q": 0}, b"null"), ({"v": 0}, b"null"), ({"q": 264}, b"aligned"),
    ({"stride": (124, 64)}, b"aligned"), ({"stride": (0, 64)}, b"positive"), ({"stride": (2 ** 38, 64)}, b"strides")])
def test_sequence_arguments(lib, change, text):
    assert lib.p3d_sequence_fwd(sequence(**change), DUMMY, None, None) == 1
    assert text in lib.p3d_last_error()
    assert lib.p3d_sequence_bwd(sequence(**change), DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, 1 << 40, None) == 1
    assert lib.p3d_sequence_bwd_workspace(sequence(**change)) == 0


def test_sequence_limits_and_pointers(lib):
    assert lib.p3d_sequence_fwd(None, DUMMY, None, None) == 1
    assert lib.p3d_sequence_fwd(sequence(q_rows=2 ** 30), DUMMY, None, None) == 2
    assert lib.p3d_sequence_fwd(sequence(sequences=2 ** 24), DUMMY, None, None) == 2
    assert lib.p3d_sequence_fwd(sequence(), None, None, None) == 1 and b"output" in lib.p3d_last_error()
    assert lib.p3d_sequence_fwd(sequence(), 264, None, None) == 1
    assert lib.p3d_sequence_bwd(sequence(), DUMMY, None, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, 1 << 40, None) == 1
    assert lib.p3d_sequence_bwd(sequence(), DUMMY, DUMMY, DUMMY, 264, DUMMY, DUMMY, DUMMY, 1 << 40, None) == 1
    assert lib.p3d_sequence_fwd(sequence(q_rows=0, q=0), None, None, None) == 0      # nothing to do


@pytest.mark.parametrize("change,text", [
    ({"dtype": 7}, b"dtype"), ({"dim": 60}, b"multiple of 8"), ({"dim": 264}, b"multiple of 8"), ({"heads": 0}, b"positive"),
    ({"page": 0}, b"positive"), ({"pages": 0}, b"positive"), ({"pages": 2 ** 31}, b"at most"), ({"sequences": -1}, b"negative"),
    ({"width": 2 ** 28}, b"places"), ({"k": 0}, b"given"), ({"v": 264}, b"aligned"), ({"dtype": 3}, b"scales"), ({"table": 0}, b"table")])
def test_cache_arguments(lib, change, text):
    strides = PAIR.pack(64, 64)
    append = lib.p3d_cache_append(cache(**change), DUMMY, strides, DUMMY, strides, 2, 4, DUMMY, DUMMY, None)
    assert append == 1 and text in lib.p3d_last_error()
    assert lib.p3d_cache_read(cache(**change), None, DUMMY, 4, DUMMY, DUMMY, 2, None) == 1
    assert lib.p3d_paged_attention(cache(**change), DUMMY, strides, 2, 2, DUMMY, 0.1, DUMMY, None, 0, None) == 1
    assert lib.p3d_paged_attention_workspace(cache(**change), 2) == 0


def test_cache_limits_and_pointers(lib):
    strides = PAIR.pack(64, 64)
    append = lambda c, k=DUMMY, s=strides, dtype=2, rows=4, starts=DUMMY: lib.p3d_cache_append(c, k, s, DUMMY, strides, dtype, rows, starts,  # noqa: E731
                                                                                             DUMMY, None)
    assert append(cache(), dtype=1) == 1 and b"dtype" in lib.p3d_last_error()
    assert append(cache(), rows=-1) == 1 and append(cache(), rows=2 ** 31) == 1
    assert append(cache(), k=None) == 1 and append(cache(), starts=None) == 1
    assert append(cache(), k=264) == 1 and append(cache(), s=PAIR.pack(60, 64)) == 1
    assert append(cache(), rows=0) == 0 and append(cache(sequences=0)) == 0
    assert lib.p3d_cache_read(cache(), None, DUMMY, 4, DUMMY, None, 2, None) == 1
    assert lib.p3d_cache_read(cache(), None, DUMMY, 4, DUMMY, DUMMY, 3, None) == 1
    assert lib.p3d_cache_read(cache(sequences=0), None, DUMMY, 4, DUMMY, DUMMY, 2, None) == 1
    assert lib.p3d_cache_read(cache(), None, None, 0, None, None, 2, None) == 0
    attend = lambda c, heads=2, dtype=2, scale=0.1, q=DUMMY: lib.p3d_paged_attention(c, q, strides, dtype, heads, DUMMY, scale, DUMMY, None, 0, None)  # noqa: E731
    assert attend(cache(dim=136)) == 1 and attend(cache(heads=2), heads=3) == 1 and attend(cache(), dtype=0) == 1
    assert attend(cache(), dtype=1) == 1 and attend(cache(), scale=-1.0) == 1 and attend(cache(), q=None) == 1
    assert attend(cache(pages=2 ** 30, heads=16, page=64), heads=16) == 2
    assert attend(cache(sequences=0)) == 0


def test_cpu_tensors_are_refused_not_computed():
    from pack3d_b200 import PagedCache, norm_rotate, paged_attention, sequence_attention
    x, o = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    pages = PagedCache(2, 2, 8, 64, device="cpu")
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: norm_rotate(x, None, torch.arange(4)), lambda: sequence_attention(x, x, x, o),
                 lambda: pages.append(x, x, table, lengths, o), lambda: pages.read(table, o, 4),
                 lambda: paged_attention(x[:1], pages, table, lengths)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_tangents_are_refused():
    import torch.autograd.forward_ad as forward_ad
    from pack3d_b200 import norm_rotate, sequence_attention
    x, o = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        for call in (lambda: norm_rotate(dual, None, torch.arange(4)), lambda: sequence_attention(x, dual, x, o)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_cache_shapes_are_checked():
    from pack3d_b200 import PagedCache
    for bad in ((0, 1, 1, 8), (1, 0, 1, 8), (1, 1, 0, 8), (1, 1, 1, 12), (1, 1, 1, 264), (True, 1, 1, 8), (1.0, 1, 1, 8)):
        with pytest.raises(ValueError):
            PagedCache(*bad, device="cpu")
    cache8 = PagedCache(3, 2, 4, 16, dtype=torch.float8_e4m3fn, device="cpu")
    assert cache8.k.shape == (3, 2, 4, 16) and cache8.k_scales.shape == (3, 2, 4) and cache8.page_size == 4
    assert cache8.dtype is torch.float8_e4m3fn and (cache8.v_scales == 127).all()
    assert PagedCache(1, 1, 1, 8, device="cpu").k_scales is None


def test_host_module_has_the_operators():
    from pack3d_b200 import _native
    module = _native.host()
    assert {"norm_rotate", "sequence_attention", "cache_append", "cache_read", "paged_attention"} <= set(dir(module))
    with pytest.raises(ValueError, match="takes"):
        module.norm_rotate(torch.zeros(2))
    assert ctypes.sizeof(ctypes.c_void_p) == 8
