"""What the header promises of the 8-bit cache's calls beside their shapes, without a GPU."""

import ctypes
import re

import numpy as np
import pytest

from qdec import capi
from test_kv8_capi import attn, merging, one


@pytest.mark.parametrize("nq,nkv,t,d", [(40, 8, 1, 128), (40, 8, 3, 128), (9, 3, 5, 64), (8, 8, 1, 128), (30, 10, 1, 64), (32, 8, 1, 128)])
def test_partials_begin_on_16_bytes(qlib, nq, nkv, t, d):
    """A split's partial of an odd number of rows R takes R (head_dim + 2) + 2 floats."""
    r = t * nq // nkv
    one = 4 * (r * (d + 2) + (2 if r % 2 else 0))
    assert one % 16 == 0
    for splits in (2, 3, 7):
        assert qlib.kv8_attn_workspace(attn(nq=nq, nkv=nkv, t_rows=t, head_dim=d, splits=splits)) == (2 * nkv * splits * one, 0)


@pytest.mark.parametrize("at,kw,code,needle", [
    ({}, dict(x_frag=1), -3, "x_frag needs no"),
    (dict(batch=4), dict(rows=4, x_frag=1), -3, "x_frag needs no"),
    (dict(batch=17), dict(rows=17, waves=4, x_frag=1), -3, "x_frag needs no"),
    ({}, dict(flags=capi.GLU, x_frag=1), -3, "x_frag needs no"),
    ({}, dict(flags=capi.ARGMAX, x_frag=1), -3, "x_frag needs no"),
    ({}, dict(x_parts=16, x_nparts=2, x_merged=32), -3, "x_parts needs"),
    ({}, dict(x_parts=16, x_nparts=2, x_merged=32, flags=capi.NORM_IN), -3, "x_parts needs"),
    ({}, dict(flags=capi.NORM_IN), -3, "NORM_IN"),
    (dict(out_partials=0), {}, -1, "out_partials"),
    (dict(nq=64), dict(k=8192), -1, "shape"),
    (dict(batch=2), {}, -1, "rows 1"),
    (dict(lens=None), {}, -1, "lens"),
    ({}, dict(resident=1), -3, "resident"),
    ({}, dict(ksplit=2), -3, "registers"),
])
def test_a_product_names_the_partials_it_refuses(qlib, at, kw, code, needle):
    """The partials of an 8-bit call are refused where those of a bf16 call are, by their own name."""
    a = one(**at)
    g = merging(a, **kw)
    assert qlib.so.qdec_gemm(ctypes.byref(g), None) == code
    assert needle in qlib.last_error() and "x_kv8" in qlib.last_error()


def test_a_many_row_product_takes_no_partials(qlib):
    a = one(batch=16)
    g = merging(a, rows=16, waves=4)
    assert qlib.so.qdec_gemm_wide_workspace(ctypes.byref(g), None) == -3 and "x_kv8" in qlib.last_error()


def test_a_library_tells_its_structs_sizes(qlib):
    """Every argument struct of the header is mirrored and has the library's size, and a
    caller with another one can tell before it calls."""
    text = re.sub(r"/\*.*?\*/", "", open(capi.HEADER).read(), flags=re.S)
    assert sorted(re.findall(r"\}\s*(qdec_\w+_args);", text)) == sorted(capi.ARGS)
    for name, st in capi.ARGS.items():
        assert qlib.so.qdec_args_size(name.encode()) == ctypes.sizeof(st), name
    for name in (b"qdec_gem_args", b"", None):
        assert qlib.so.qdec_args_size(name) == -1 and "struct" in qlib.last_error()


def test_a_binding_of_another_header_is_refused(monkeypatch):
    class Shorter(ctypes.Structure):  # the product's arguments before x_kv8
        _fields_ = [f for f in capi.GemmArgs._fields_ if f[0] != "x_kv8"]

    assert ctypes.sizeof(Shorter) < ctypes.sizeof(capi.GemmArgs)
    monkeypatch.setitem(capi.ARGS, "qdec_gemm_args", Shorter)
    with pytest.raises(RuntimeError, match="qdec_gemm_args"):
        capi.Lib()


def test_quotients_near_a_half():
    """127 x / top of bf16 numbers 2^7 <= X, T < 2^8, x / top = X / T 2^-k: a half, or further
    from one than 2^-16 of itself, which the kernels' fp32 quotient (within 2^-23) tells
    apart.  From k = 9 on it is below 0.495."""
    X, T = np.meshgrid(np.arange(128, 256), np.arange(128, 256))
    least = 1.0
    for k in range(9):
        num, den = 254 * X, (T << k)  # twice the quotient, which is odd where it is a half
        held = X <= den
        off = np.abs(num - (num // (2 * den) * 2 + 1) * den)  # to the half above the whole number below
        held &= off > 0
        least = min(least, (off[held] / num[held]).min())
    assert 2.0 ** -16 < least < 2.0 ** -15.9
    assert 127 * 255 / (128 * 2 ** 9) < 0.495


def test_splits_of_the_longest_cache(qlib):
    """The chosen number follows the cap up to the largest there is."""
    got = [qlib.kv8_attn_workspace(attn(batch=2, nkv=1, nq=4, t_rows=1, cap=cap))[0] // (2 * 4 * 4 * 130)
           for cap in (1 << 20, (1 << 31) - 1024, (1 << 31) - 512, (1 << 31) - 256, (1 << 31) - 64)]
    assert got == [128] * 5
