"""The 8-bit KV cache restated in 64 bits, slot by slot.

A row x is held as q = round(127 x / max|x|), ties to even, and scale = max|x| /
127; rows whose maximum is below 2^-100 as zeros with scale 0, rows with an
infinity or a NaN as q = 0 with scale NaN.  Caches: K [nkv, cap, D] and V [nkv,
cap/16, D, 16] int8 per sequence, scales [nkv, cap]."""

import math

import torch

TINY = 2.0 ** -100


def hold(x):
    """(q, scale) of rows [..., D] in 64 bits, q whole numbers."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    q = torch.round(127 * x / top.clamp(min=TINY))
    scale = top / 127
    q = torch.where(top < TINY, 0.0, q)
    scale = torch.where(top < TINY, 0.0, scale)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    return torch.where(bad, 0.0, q), torch.where(bad, math.nan, scale)[..., 0]


def row_major(v8):
    """V [..., cap/16, D, 16] as [..., cap, D]."""
    return v8.transpose(-1, -2).flatten(-3, -2)


def slab_rows(v):
    """A V slab [..., cap/8, D, 8] as [..., cap, D]."""
    return v.transpose(-1, -2).flatten(-3, -2)


def norm_rope(x, w, cos, sin, eps):
    """Head RMSNorm and RoPE of rows [T, heads, D] at positions of cos, sin [T, D]."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    half = x.shape[-1] // 2
    rot = torch.cat((-y[..., half:], y[..., :half]), -1)
    return y * cos.double()[:, None] + rot * sin.double()[:, None]


def attend(q, k8, ks, v8, vs, L, scale):
    """Rows q [T, nq, D] (row t at position L + t) over the cache of one
    sequence that already holds slots up to L + T - 1.  Returns (out [T, nq,
    D], mag: sum |p v| / sum p, step: 128 n max(p v_scale) / sum p [T, nq, 1],
    reach and grid: max sum |q k| * scale and max|q| * sum |k| * scale over seen slots)."""
    T, nq, D = q.shape
    nkv = k8.shape[0]
    G = nq // nkv
    out = torch.zeros_like(q)
    mag = torch.zeros_like(q)
    step = torch.zeros_like(q[..., :1])
    reach = grid = 0.0
    keys = k8[:, :L + T].double() * ks[:, :L + T, None].double()
    vals = row_major(v8.double())[:, :L + T] * vs[:, :L + T, None].double()
    for t in range(T):
        n = L + t + 1
        for h in range(nkv):
            qh = q[t, h * G:(h + 1) * G]
            p = torch.softmax(qh @ keys[h, :n].t() * scale, -1)
            out[t, h * G:(h + 1) * G] = p @ vals[h, :n]
            mag[t, h * G:(h + 1) * G] = p @ vals[h, :n].abs()
            step[t, h * G:(h + 1) * G] = 128 * n * (p * vs[h, :n].double()).amax(-1, keepdim=True)
            size = keys[h, :n].abs()
            r = float((qh.abs() @ size.t()).max() * scale)
            reach = max(reach, r) if math.isfinite(r) else reach
            r = float(qh.abs().max() * size.sum(-1).max() * scale)
            grid = max(grid, r) if math.isfinite(r) else grid
    return out, mag, step, reach, grid
