"""Refusals of the tree attention that come before any HIP call."""

import pytest
from test_tree_capi import attn

from qdec import capi


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), -float("inf"), 1e-40])
def test_attention_scale(qlib, scale):
    """The scores' scale is positive, and neither it nor its reciprocal leaves
    fp32's range (no launch happens: the refusal is the first to apply)."""
    with pytest.raises(capi.QdecError, match="sm_scale"):
        qlib.tree_attn(attn(sm_scale=scale), None)
    qlib.tree_attn_workspace(attn(sm_scale=scale))  # does not need it


@pytest.mark.parametrize("kw", [dict(batch=65535, splits=33), dict(batch=65535, splits=256),
                                dict(batch=1024, nkv=2048, nq=2048, splits=16),
                                dict(batch=4, nkv=65535, nq=65535, t_rows=64, splits=33),
                                dict(batch=65535, nkv=64, nq=256, t_rows=64, splits=2)])  # in the merge
def test_attention_more_work_items_than_a_launch_numbers(qlib, kw):
    """2^32 work items or more in one launch: 256 a workgroup, one workgroup per
    sequence, kv head, row group and split."""
    a = attn(**kw)
    with pytest.raises(capi.QdecError, match="row groups"):
        qlib.tree_attn_workspace(a)
    with pytest.raises(capi.QdecError, match="row groups"):
        qlib.tree_attn(a, None)


@pytest.mark.parametrize("kw", [dict(batch=65535, splits=31), dict(batch=2, splits=256), dict(batch=64, t_rows=64, splits=16)])
def test_attention_workspace_below_that(qlib, kw):
    assert qlib.tree_attn_workspace(attn(**kw))[0] > 0
