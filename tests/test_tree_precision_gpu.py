"""How precise the tree attention is: queries in two bf16 parts where few rows share
a workgroup, rounded once where many do, each against its own 64-bit definition;
and a chain's outputs beside the decode attention's."""

import pytest
import torch
from test_tree_gpu import DEV, EPS, NAN, Attn, lib, rope, stream, v_layout  # noqa: F401  (lib: the fixture)
from tree_contests import SHAPES, L, bound, inputs, near_a_tie, reference

from oracle import tree_oracle
from qdec import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,nq,nkv,D,cap,rows", SHAPES)
@pytest.mark.parametrize("splits", [0, 2])
def test_queries(lib, B, T, nq, nkv, D, cap, rows, splits):  # noqa: F811
    x = inputs(B, T, nq, nkv, D, cap, seed=T)
    c = Attn(lib, [L] * B, T, nq, nkv, D, "star", splits=splits, cap=cap)
    a = capi.TreeAttnArgs.from_buffer_copy(c.a)
    a.splits = 2
    groups = -(-T * (nq // nkv) // rows)
    assert lib.tree_attn_workspace(a)[0] == 4 * B * nkv * 2 * groups * rows * (D + 2)
    k, v = x["k"].clone(), x["v"].clone()
    k[:, :, L:] = NAN
    v[:, :, L:] = NAN
    for dst, src in ((c.qkv, x["qkv"]), (c.qn, x["qn"]), (c.kn, x["kn"]), (c.cos, x["cos"]), (c.sin, x["sin"]), (c.k, k),
                     (c.v, v_layout(v))):
        dst.copy_(src)
    c.run()
    torch.cuda.synchronize()
    got = c.rows().double().cpu()
    wide = rows >= 128
    for b in range(B):
        out, mag, _, _ = reference(x, b, nq, nkv, tree_oracle.bf if wide else lambda q: q)
        limit = bound(x, b, nq, nkv, out, mag)
        if wide:
            limit[near_a_tie(x, b, nq, nkv)] = float("inf")
        worst = ((got[b] - out).abs() / limit).max().item()
        assert worst <= 1, (b, worst)


def test_chain_outputs_against_the_decode_attention(lib):  # noqa: F811
    """A chain through qdec_attn and through qdec_tree_attn.  qdec_attn rounds a
    normalised, rotated entry at most five times, each by 2^-8 of its two terms,
    and the probabilities once; the tree rounds once each at most.  So a score
    differs by at most 12 * 2^-8 of sum |q k| / sqrt(D), where |q| <= sqrt(2 D)
    max|gain| (the terms' norm) and |k| alike, and an output by twice that
    (numerator and denominator), 2 * 2^-8 for the probabilities, all of mag, and
    both roundings.  Independent roundings of a score of rms 1 add up to
    sqrt(10 / 3) * 2^-8 = 0.0071, twice that in an output: the mean difference is
    below 2^-5 of mag."""
    B, T, nq, nkv, D, cap = 3, 8, 32, 8, 128, 640
    lens = [0, 333, 600]
    c = Attn(lib, lens, T, nq, nkv, D, "chain", cap=cap, seed=2)
    c.qkv.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    c.cos, c.sin = rope(cap, D)
    c.a.cos_tab, c.a.sin_tab = c.cos.data_ptr(), c.sin.data_ptr()
    c.run()
    k, v = c.k.clone(), c.v.clone()
    out = torch.zeros((B * T, nq * D), dtype=torch.bfloat16, device=DEV)
    a = capi.AttnArgs(eps=EPS, sm_scale=D ** -0.5, batch=B, t_rows=T, nq=nq, nkv=nkv, head_dim=D, cap=cap, chunk=cap,
                      waves=4)
    for f, t in (("qkv", c.qkv), ("q_norm_w", c.qn), ("k_norm_w", c.kn), ("cos_tab", c.cos), ("sin_tab", c.sin),
                 ("lens", c.lens), ("k_cache", k), ("v_cache", v), ("out", out)):
        setattr(a, f, t.data_ptr())
    lib.attn(a, stream())
    torch.cuda.synchronize()
    for b, L in enumerate(lens):
        ref, mag, kn, _ = tree_oracle.attention(c.qkv[b * T:(b + 1) * T], c.trees[b], L, c.k[b], c.v_rows[b], c.qn,
                                                c.kn, c.cos, c.sin, nq, nkv, EPS)
        got, dec = c.rows()[b].double(), out.view(B, T, nq, D)[b].double()
        gain = float(c.qn.double().abs().max())
        kmax = max(float(kn.abs().max()), float(c.k[b, :, :L].double().abs().max()) if L else 0.0)
        score = 12 * 2.0 ** -8 * 2 * D ** 0.5 * gain * kmax
        limit = 2 * ref.abs() * 2.0 ** -8 + mag * (2 * score + 2 * 2.0 ** -8)
        diff = (got - dec).abs()
        assert (diff <= limit).all() and diff.mean() <= mag.mean() * 2.0 ** -5, (b, diff.mean(), mag.mean())
