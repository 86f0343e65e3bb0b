"""Inputs of the tree attention on which a query's rounding shows, shared by the
tests on the CPU and on the GPU.

Every cached key has four channels that are not zero, with scores of standard
deviation 16, so that some rows' first two slots are close.  Rounding a
query's entries to bf16 moves a score by about 2^-8 / sqrt(6) * 16 = 0.026, and
the output of a close row by that part of the values.  What the kernels may be
off is far less, by ``bound``.  Node keys are short: their weight is nothing."""

import torch

from oracle import tree_oracle

EPS = 1e-6
L = 40


def inputs(B, T, nq, nkv, D, cap, seed):
    """Host tensors of B sequences of L cached slots, a star of T nodes each."""
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g)

    k = torch.zeros((B, nkv, cap, D))
    at = torch.rand((B, nkv, L, D), generator=g).topk(4, -1).indices
    k[:, :, :L].scatter_(3, at, normal(B, nkv, L, 4) * (16 * D ** 0.5 / 2))
    v = torch.zeros((B, nkv, cap, D))
    v[:, :, :L] = normal(B, nkv, L, D)
    inv = 1.0 / (1e4 ** (torch.arange(0, D, 2, dtype=torch.float32) / D))
    ang = torch.arange(cap, dtype=torch.float32)[:, None] * inv
    ang = torch.cat((ang, ang), 1)
    x = dict(qkv=normal(B * T, (nq + 2 * nkv) * D), qn=1 + 0.2 * normal(D), kn=0.01 * normal(D), cos=ang.cos(),
             sin=ang.sin(), k=k, v=v)
    x = {n: t.to(torch.bfloat16) for n, t in x.items()}
    x["parents"] = [-1] + [0] * (T - 1)
    return x


def reference(x, b, nq, nkv, round_q):
    T = len(x["parents"])
    return tree_oracle.attention(x["qkv"][b * T:(b + 1) * T], x["parents"], L, x["k"][b], x["v"][b], x["qn"], x["kn"],
                                 x["cos"], x["sin"], nq, nkv, EPS, round_q)


def bound(x, b, nq, nkv, out, mag):
    """[T, nq, D]: what an output may be off where its query is not rounded.  A
    score: relative to sum |q k| / sqrt(D), with |q| the sum of its rotation's two
    terms, 2^-16 for a query in two bf16 parts, 256 * 2^-24 for the fp32 sum of two
    products of 128, 2^-19 for the fp32 norm and rotation, and 2^-22 for its place
    in the exponent.  The output: twice that of mag (numerator and denominator),
    2^-16 for the probabilities' two parts, the fp32 sums over the rows, and its own
    rounding."""
    T, D = len(x["parents"]), x["cos"].shape[1]
    q, terms = queries(x, b, nq, nkv)
    kc = x["k"][b, :, :L].double()
    s = torch.matmul(terms.view(T, nkv, nq // nkv, D).permute(1, 0, 2, 3).reshape(nkv, -1, D),
                     kc.abs().transpose(1, 2).contiguous()).amax(-1) / D ** 0.5
    s = s.view(nkv, T, nq // nkv).permute(1, 0, 2).reshape(T, nq, 1)
    score = s * (2.0 ** -16 + 2.0 ** -16 + 2.0 ** -19 + 2.0 ** -22)
    return out.abs() * 2.0 ** -8 + mag * (2 * score + 2.0 ** -16 + (L + T + 64) * 2.0 ** -22)


def queries(x, b, nq, nkv):
    """Queries [T, nq, D] and the sum of the absolute values of the two terms of
    each of their entries, in 64 bits."""
    T, D = len(x["parents"]), x["cos"].shape[1]
    y = x["qkv"][b * T:(b + 1) * T].double().view(T, -1, D)[:, :nq]
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * x["qn"].double()
    pos = torch.tensor([L] + [L + 1] * (T - 1))
    c, s = x["cos"][pos][:, None].double(), x["sin"][pos][:, None].double()
    half = torch.cat((-y[..., D // 2:], y[..., :D // 2]), -1)
    return y * c + half * s, (y * c).abs() + (half * s).abs()


def near_a_tie(x, b, nq, nkv):
    """[T, nq]: some entry of the query is so near to half way between two bf16
    values that fp32 arithmetic may round it to the other one."""
    q, terms = queries(x, b, nq, nkv)
    step = 2.0 ** (torch.floor(torch.log2(q.abs().clamp(min=1e-30))) - 7)
    off = ((q.abs() / step) % 1 - 0.5).abs() * step
    return (off <= terms * 2.0 ** -19).any(-1)


# B, T, nq, nkv, D, cap, rows of a group: the narrow kernel with one and two
# tiles, the wide one with 4 and 8 waves
SHAPES = [(3, 4, 8, 2, 128, 96, 16), (3, 5, 6, 2, 64, 96, 16), (8, 8, 32, 8, 128, 96, 32), (16, 16, 16, 4, 64, 96, 32),
          (1, 27, 32, 8, 128, 12256, 128), (1, 20, 64, 8, 128, 10304, 256), (1, 9, 32, 2, 64, 82016, 256)]
