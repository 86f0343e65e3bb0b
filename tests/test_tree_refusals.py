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
