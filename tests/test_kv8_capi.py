"""The 8-bit cache's entry points without a GPU: argument structs that mirror the
header, refusals before any HIP call, workspace sizes; and the oracle."""

import ctypes
import math
import re

import pytest
import torch

from oracle import kv8_oracle
from qdec import capi


def test_structs_match_header_fields():
    text = re.sub(r"/\*.*?\*/", "", open(capi.HEADER).read(), flags=re.S)
    for cname, st in (("qdec_kv8_store_args", capi.Kv8StoreArgs), ("qdec_kv8_load_args", capi.Kv8LoadArgs),
                      ("qdec_kv8_attn_args", capi.Kv8AttnArgs)):
        body = re.search(r"typedef struct(?: \w+)? \{([^{}]*)\}\s*" + cname + ";", text).group(1)
        assert re.findall(r"\*?\s*(\w+)\s*;", body) == [f[0] for f in st._fields_], cname


def fill(st, **kw):
    a = st()
    for f, t in a._fields_:
        setattr(a, f, 16 if t is capi.P else 1)  # (eps and sm_scale: 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def store(**kw):
    return fill(capi.Kv8StoreArgs, **{**dict(batch=2, nkv=8, head_dim=128, cap=1024, slab_cap=512, pos0=3, n=100), **kw})


def load(**kw):
    return fill(capi.Kv8LoadArgs, **{**dict(batch=2, nkv=8, head_dim=128, cap=1024, slab_cap=512, n=100), **kw})


def attn(**kw):
    return fill(capi.Kv8AttnArgs, **{**dict(batch=2, t_rows=4, nq=32, nkv=8, head_dim=128, cap=1024, splits=0,
                                            out_frag=0, out_partials=0), **kw})


def shared(name, make):
    return [
        (name, make, dict(head_dim=96), -3, "head_dim"),
        (name, make, dict(batch=0), -1, "batch"),
        (name, make, dict(batch=16384), -1, "batch"),
        (name, make, dict(nkv=0), -1, "nkv"),
        (name, make, dict(cap=0), -1, "cap"),
        (name, make, dict(cap=1056), -1, "multiple of 64"),
        (name, make, dict(k8=None), -1, "null"),
        (name, make, dict(v8=None), -1, "null"),
        (name, make, dict(k_scale=None), -1, "null"),
        (name, make, dict(v_scale=None), -1, "null"),
        (name, make, dict(k8=24), -2, "aligned"),
        (name, make, dict(v8=8), -2, "aligned"),
        (name, make, dict(v_scale=4), -2, "aligned"),
    ]


CASES = shared("kv8_store", store) + shared("kv8_load", load) + shared("kv8_attn", attn) + [
    ("kv8_store", store, dict(slab_cap=0), -1, "slab_cap"),
    ("kv8_store", store, dict(slab_cap=520), -1, "multiple of 32"),
    ("kv8_store", store, dict(pos0=-1), -1, "slots"),
    ("kv8_store", store, dict(n=0), -1, "slots"),
    ("kv8_store", store, dict(pos0=500), -1, "slots"),
    ("kv8_store", store, dict(pos0=2147483600, n=100), -1, "slots"),
    ("kv8_store", store, dict(slab_cap=2048, pos0=1000), -1, "slots"),
    ("kv8_store", store, dict(k_slab=None), -1, "null"),
    ("kv8_store", store, dict(v_slab=8), -2, "aligned"),
    ("kv8_store", store, dict(batch=16383, nkv=65535), -3, "pairs"),
    ("kv8_load", load, dict(slab_cap=48), -1, "slab_cap"),
    ("kv8_load", load, dict(n=0), -1, "n 0"),
    ("kv8_load", load, dict(n=513), -1, "n 513"),
    ("kv8_load", load, dict(v_slab=None), -1, "null"),
    ("kv8_load", load, dict(k_slab=8), -2, "aligned"),
    ("kv8_load", load, dict(batch=16383, nkv=65535), -3, "pairs"),
    ("kv8_attn", attn, dict(nq=30), -3, "nq"),
    ("kv8_attn", attn, dict(nq=4), -3, "nq"),
    ("kv8_attn", attn, dict(t_rows=0), -1, "t_rows"),
    ("kv8_attn", attn, dict(t_rows=17), -1, "t_rows"),
    ("kv8_attn", attn, dict(t_rows=9, nq=64), -3, "64 rows"),
    ("kv8_attn", attn, dict(sm_scale=0.0), -1, "sm_scale"),
    ("kv8_attn", attn, dict(sm_scale=-0.1), -1, "sm_scale"),
    ("kv8_attn", attn, dict(sm_scale=math.inf), -1, "sm_scale"),
    ("kv8_attn", attn, dict(sm_scale=math.nan), -1, "sm_scale"),
    ("kv8_attn", attn, dict(splits=-1), -1, "splits"),
    ("kv8_attn", attn, dict(splits=257), -1, "splits"),
    ("kv8_attn", attn, dict(out_frag=2), -1, "out_frag"),
    ("kv8_attn", attn, dict(out_partials=2), -1, "out_partials"),
    ("kv8_attn", attn, dict(out_partials=1, splits=1, partial=None), -1, "partial"),
    ("kv8_attn", attn, dict(batch=16383, nkv=1000, nq=4000, splits=2), -3, "splits"),
    ("kv8_attn", attn, dict(splits=2, partial=None), -1, "partial"),
    ("kv8_attn", attn, dict(splits=2, partial=8), -2, "aligned"),
    ("kv8_attn", attn, dict(qkv=8), -2, "aligned"),
    ("kv8_attn", attn, dict(cos_tab=24), -2, "aligned"),
    ("kv8_attn", attn, dict(out=24), -2, "aligned"),
] + [("kv8_attn", attn, {f: None}, -1, "null") for f in ("qkv", "q_norm_w", "k_norm_w", "cos_tab", "sin_tab", "lens", "out")]


@pytest.mark.parametrize("name,make,kw,code,needle", CASES, ids=[f"{c[0]}-{c[2]}" for c in CASES])
def test_refusals(qlib, name, make, kw, code, needle):
    a = make(**kw)
    assert getattr(qlib.so, "qdec_" + name)(ctypes.byref(a), None) == code
    assert needle in qlib.last_error()
    with pytest.raises(capi.QdecError):
        getattr(qlib, name)(a, None)


@pytest.mark.parametrize("name", ["kv8_store", "kv8_load", "kv8_attn"])
def test_null_args(qlib, name):
    assert getattr(qlib.so, "qdec_" + name)(None, None) == -1


def merging(at, **kw):
    """An O projection that merges the attention call's partials."""
    g = fill(capi.GemmArgs, **{**dict(rows=1, n=2560, k=4096, flags=capi.RES_OUT, waves=8, x=None, x_attn=None, parts_out=None,
                                      x_parts=None, x_frag=0, out_frag=0, next_norm_w=None, resident=0), **kw})
    g.x_kv8 = ctypes.addressof(at)
    return g


def one(**kw):
    return attn(**{**dict(batch=1, t_rows=1, out_partials=1), **kw})


def test_merge_in_a_gemm(qlib):
    for at, kw in ((one(), {}), (one(splits=1), {}), (one(cap=1 << 20), {}), (one(batch=2), dict(rows=2)),
                   (one(nq=16, nkv=4), dict(k=2048))):
        qlib.gemm_workspace(merging(at, **kw))


@pytest.mark.parametrize("at,kw,code,needle", [
    (dict(out_partials=0), {}, -1, "out_partials"),
    (dict(nq=64), dict(k=8192), -1, "shape"),
    (dict(nq=16), dict(k=2048), -1, "shape"),
    (dict(head_dim=64, nq=32), dict(k=2048), -1, "shape"),
    (dict(cap=0), {}, -1, "shape"),
    (dict(splits=-1), {}, -1, "shape"),
    (dict(splits=257), {}, -1, "shape"),
    (dict(batch=0), {}, -1, "shape"),
    (dict(t_rows=2), dict(rows=2), -1, "shape"),
    (dict(batch=2), {}, -1, "rows 1"),
    ({}, dict(k=2048), -1, "rows 1"),
    ({}, dict(flags=capi.NORM_IN), -3, "NORM_IN"),
    ({}, dict(x_attn=16), -1, "both"),
    ({}, dict(resident=1), -3, "x_attn"),
    ({}, dict(ksplit=2, k=4096), -3, "x_attn"),
    (dict(batch=5), dict(rows=5), -3, "x_attn"),
    (dict(partial=None), {}, -1, "partial"),
    (dict(lens=None), {}, -1, "lens"),
])
def test_merge_refusals(qlib, at, kw, code, needle):
    a = one(**at)
    g = merging(a, **kw)
    assert qlib.so.qdec_gemm(ctypes.byref(g), None) == code
    assert needle in qlib.last_error()


def test_workspace(qlib):
    assert qlib.kv8_attn_workspace(attn(splits=1)) == (0, 0)
    assert qlib.kv8_attn_workspace(attn(splits=1, out_partials=1)) == (4 * 2 * 4 * 32 * 130, 0)
    for nq, t, d, s in ((32, 4, 128, 2), (8, 16, 64, 7), (64, 8, 128, 256)):
        assert qlib.kv8_attn_workspace(attn(splits=s, nq=nq, t_rows=t, head_dim=d)) == (4 * 2 * t * nq * s * (d + 2), 0)
    # splits = 0 follows from batch, nkv and cap alone
    assert qlib.kv8_attn_workspace(attn(batch=1, cap=64)) == (0, 0)
    big = [qlib.kv8_attn_workspace(attn(batch=1, cap=1 << 20, t_rows=t, nq=nq))[0] // (4 * t * nq * 130)
           for t, nq in ((1, 32), (4, 32), (1, 64), (16, 8))]
    assert big[0] > 1 and len(set(big)) == 1


def test_oracle_holds_rows():
    x = torch.tensor([[1.0, -2.0, 0.5, 1.5], [0.0, 0.0, 0.0, 0.0], [2.0 ** -101, 0, 0, 0], [1.0, math.inf, 0, 0],
                      [math.nan, 1, 2, 3], [254.0, 3.0, 5.0, -1.0]])
    q, s = kv8_oracle.hold(x)
    # 63.5 and 31.75 and 95.25; 127 * 3 / 254 = 1.5 and 127 * 5 / 254 = 2.5 go to the even neighbour
    assert q.tolist() == [[64, -127, 32, 95], [0] * 4, [0] * 4, [0] * 4, [0] * 4, [127, 2, 2, 0]]
    assert s[0] == 2 / 127 and s[1] == 0 and s[2] == 0 and torch.isnan(s[3]) and torch.isnan(s[4]) and s[5] == 2


def test_oracle_attends():
    """One head, two slots, by hand."""
    D = 64
    k8 = torch.zeros((1, 64, D), dtype=torch.int8)
    v8 = torch.zeros((1, 4, D, 16), dtype=torch.int8)
    k8[0, 0, 0], k8[0, 1, 0] = 10, -10
    v8[0, 0, :, 0], v8[0, 0, :, 1] = 3, 5
    ks, vs = torch.zeros((1, 64)), torch.zeros((1, 64))
    ks[0, :2], vs[0, :2] = 0.1, 2.0
    q = torch.zeros((1, 1, D), dtype=torch.float64)
    q[0, 0, 0] = 2.0
    out, mag, step, reach, grid = kv8_oracle.attend(q, k8, ks, v8, vs, 1, 0.5)
    w = math.exp(-2.0)
    assert torch.allclose(out, torch.full_like(out, (6 + 10 * w) / (1 + w)), rtol=1e-6)
    assert abs(step[0, 0, 0].item() - 128 * 2 * 2 / (1 + w)) < 1e-4
    assert torch.equal(out, mag) and abs(reach - 1.0) < 1e-6 and abs(grid - 1.0) < 1e-6
