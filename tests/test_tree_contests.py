"""The inputs that pin the queries' precision do so: with queries rounded to
bf16, all of them or one k step's (32 channels), the 64-bit result leaves the
bound, in every tile of 16 query rows."""

import pytest
import torch
from tree_contests import L, SHAPES, bound, inputs, near_a_tie, reference

from oracle.tree_oracle import bf


@pytest.mark.parametrize("B,T,nq,nkv,D,cap,rows", SHAPES)
def test_a_rounded_query_shows(B, T, nq, nkv, D, cap, rows):
    x = inputs(B, T, nq, nkv, D, min(cap, 96), seed=T)
    G, steps = nq // nkv, D // 32
    tile = (torch.arange(T)[:, None] * G + torch.arange(nq)[None] % G) // 16  # a query row's, among its kv head's
    shown = torch.zeros((steps + 1, int(tile.max()) + 1), dtype=torch.int64)
    kept = total = 0
    for b in range(B):
        out, mag, _, _ = reference(x, b, nq, nkv, lambda q: q)
        limit = bound(x, b, nq, nkv, out, mag)
        for s in range(steps + 1):  # the last one: all channels

            def round_q(q):
                r = q.clone()
                part = slice(32 * s, 32 * s + 32) if s < steps else slice(None)
                r[..., part] = bf(q[..., part])
                return r

            bad = ((reference(x, b, nq, nkv, round_q)[0] - out).abs() > limit).any(-1)
            shown[s].index_add_(0, tile[bad], torch.ones(int(bad.sum()), dtype=torch.int64))
        clear = ~near_a_tie(x, b, nq, nkv)
        kept, total = kept + int(clear.sum()), total + clear.numel()
    assert (shown > 0).all(), shown.tolist()
    assert kept >= total / 2  # rows whose rounding is sure, for the kernel that rounds
    assert L < 96
