"""The tree entry points without a GPU: argument structs that mirror the
header, refusals before any HIP call, and workspace sizes."""

import ctypes
import re

import pytest

from qdec import capi


def test_structs_match_header_fields():
    text = re.sub(r"/\*.*?\*/", "", open(capi.HEADER).read(), flags=re.S)
    for cname, st in (("qdec_tree_draft_args", capi.TreeDraftArgs), ("qdec_tree_attn_args", capi.TreeAttnArgs),
                      ("qdec_tree_accept_args", capi.TreeAcceptArgs), ("qdec_tree_commit_args", capi.TreeCommitArgs)):
        body = re.search(r"typedef struct \{([^{}]*)\}\s*" + cname + ";", text).group(1)
        assert re.findall(r"\*?\s*(\w+)\s*;", body) == [f[0] for f in st._fields_], cname
    for name in ("QDEC_TREE_MAX_T", "QDEC_TREE_MAX_MATCHES"):
        assert int(re.search(name + r" (\d+)", text).group(1)) == getattr(capi, name[5:])


def fill(st, **kw):
    a = st()
    for f, t in a._fields_:
        setattr(a, f, 16 if t is capi.P else 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def draft(**kw):
    return fill(capi.TreeDraftArgs, **{**dict(batch=2, cap=100, t_rows=8, primary=3, backoff=2, depth=4, matches=4), **kw})


def attn(**kw):
    return fill(capi.TreeAttnArgs, **{**dict(batch=2, t_rows=8, nq=32, nkv=8, head_dim=128, cap=1024, splits=0,
                                             out_frag=0), **kw})


def accept(**kw):
    return fill(capi.TreeAcceptArgs, **{**dict(batch=2, cap=100, t_rows=8, stop_len=50), **kw})


def commit(**kw):
    return fill(capi.TreeCommitArgs, **{**dict(n_layers=2, batch=2, t_rows=8, nkv=8, head_dim=128, cap=1024), **kw})


CASES = [
    ("tree_draft", draft, dict(hist=None), -1, "null"),
    ("tree_draft", draft, dict(lens=None), -1, "null"),
    ("tree_draft", draft, dict(ids=None), -1, "null"),
    ("tree_draft", draft, dict(parents=None), -1, "null"),
    ("tree_draft", draft, dict(batch=0), -1, "batch"),
    ("tree_draft", draft, dict(batch=65536), -1, "batch"),
    ("tree_draft", draft, dict(t_rows=0), -1, "t_rows"),
    ("tree_draft", draft, dict(t_rows=65), -1, "t_rows"),
    ("tree_draft", draft, dict(cap=0), -1, "cap"),
    ("tree_draft", draft, dict(primary=0), -1, "primary"),
    ("tree_draft", draft, dict(primary=65), -1, "primary"),
    ("tree_draft", draft, dict(backoff=0), -1, "backoff"),
    ("tree_draft", draft, dict(depth=0), -1, "depth"),
    ("tree_draft", draft, dict(depth=64), -1, "depth"),
    ("tree_draft", draft, dict(matches=0), -1, "matches"),
    ("tree_draft", draft, dict(matches=33), -1, "matches"),
    ("tree_attn", attn, dict(head_dim=96), -3, "head_dim"),
    ("tree_attn", attn, dict(nq=30), -3, "nq"),
    ("tree_attn", attn, dict(nq=4), -3, "nq"),
    ("tree_attn", attn, dict(nkv=0), -3, "nkv"),
    ("tree_attn", attn, dict(nq=136), -3, "query heads"),
    ("tree_attn", attn, dict(batch=0), -1, "batch"),
    ("tree_attn", attn, dict(t_rows=0), -1, "t_rows"),
    ("tree_attn", attn, dict(t_rows=65), -1, "t_rows"),
    ("tree_attn", attn, dict(cap=0), -1, "cap"),
    ("tree_attn", attn, dict(cap=1000), -1, "multiple of 32"),
    ("tree_attn", attn, dict(splits=-1), -1, "splits"),
    ("tree_attn", attn, dict(splits=257), -1, "splits"),
    ("tree_attn", attn, dict(out_frag=2), -1, "out_frag"),
    ("tree_attn", attn, dict(batch=65535, nkv=2000, nq=2000 * 16, t_rows=64, splits=256), -3, "row groups"),
    ("tree_attn", attn, dict(parents=None), -1, "null"),
    ("tree_attn", attn, dict(k_nodes=None), -1, "null"),
    ("tree_attn", attn, dict(out=None), -1, "null"),
    ("tree_attn", attn, dict(splits=2, partial=None), -1, "partial"),
    ("tree_attn", attn, dict(splits=2, partial=8), -2, "aligned"),
    ("tree_attn", attn, dict(qkv=8), -2, "aligned"),
    ("tree_attn", attn, dict(cos_tab=24), -2, "aligned"),
    ("tree_attn", attn, dict(v_nodes=18), -2, "aligned"),
    ("tree_accept", accept, dict(out_tok=None), -1, "null"),
    ("tree_accept", accept, dict(path=None), -1, "null"),
    ("tree_accept", accept, dict(lens_out=None), -1, "null"),
    ("tree_accept", accept, dict(batch=0), -1, "batch"),
    ("tree_accept", accept, dict(t_rows=65), -1, "t_rows"),
    ("tree_accept", accept, dict(cap=0), -1, "cap"),
    ("tree_commit", commit, dict(path=None), -1, "null"),
    ("tree_commit", commit, dict(v_cache=None), -1, "null"),
    ("tree_commit", commit, dict(batch=0), -1, "batch"),
    ("tree_commit", commit, dict(t_rows=0), -1, "t_rows"),
    ("tree_commit", commit, dict(head_dim=32), -3, "head_dim"),
    ("tree_commit", commit, dict(n_layers=0), -1, "n_layers"),
    ("tree_commit", commit, dict(nkv=0), -1, "nkv"),
    ("tree_commit", commit, dict(cap=40), -1, "multiple of 32"),
    ("tree_commit", commit, dict(k_nodes=8), -2, "aligned"),
]


@pytest.mark.parametrize("name,make,kw,code,needle", CASES, ids=[f"{c[0]}-{c[2]}" for c in CASES])
def test_refusals(qlib, name, make, kw, code, needle):
    a = make(**kw)
    assert getattr(qlib.so, "qdec_" + name)(ctypes.byref(a), None) == code
    assert needle in qlib.last_error()
    with pytest.raises(capi.QdecError):
        getattr(qlib, name)(a, None)


@pytest.mark.parametrize("name", ["tree_draft", "tree_attn", "tree_accept", "tree_commit"])
def test_null_args(qlib, name):
    assert getattr(qlib.so, "qdec_" + name)(None, None) == -1


def test_workspace(qlib):
    assert qlib.tree_attn_workspace(attn(splits=1)) == (0, 0)
    # a partial holds whole row groups, D + 2 floats a row; no counters
    for nq, t, d in ((32, 8, 128), (32, 1, 64), (64, 9, 128), (40, 64, 128), (8, 64, 128), (128, 64, 64)):
        pb, cb = qlib.tree_attn_workspace(attn(splits=3, nq=nq, t_rows=t, head_dim=d))
        assert cb == 0 and pb % (4 * 16 * 3 * (d + 2)) == 0 and pb >= 4 * 16 * 3 * (d + 2) * t * (nq // 8)
    # splits = 0: the shape decides, and no more than one per four blocks of the cache
    pb, cb = qlib.tree_attn_workspace(attn(batch=1, cap=128))
    assert (pb, cb) == (0, 0)
    pb, cb = qlib.tree_attn_workspace(attn(batch=1, cap=1 << 20))
    assert pb > 0 and cb == 0
