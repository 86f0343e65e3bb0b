"""CPU restatement of tree speculation -- TEST INFRASTRUCTURE ONLY (imported
by tests/ and nothing on the product path).

The rules of include/qdec.h's tree entry points, in plain Python and 64-bit
floats: ``draft`` (the tree merged from several earlier continuations),
``ancestors`` (which rows are nodes, and what each sees), ``accept`` (the walk
along the greedy picks), ``attention`` (softmax over the cache and the
ancestors) and ``speculative_greedy`` (a whole loop around any next-token
function).  No counterpart in the reference, whose speculation verifies one
chain (notes/v10/spec.py:36-224).

Pins: tests/test_tree_oracle.py.
"""

import math

import torch


def draft(hist, L, t_rows, primary, backoff, depth, matches):
    """``(ids, parents)`` of one sequence; ``hist[L]`` is the current token."""
    L = min(max(L, 0), len(hist) - 1)
    ids, parents = [hist[L]], [-1]
    for n in (primary, backoff):
        if L < n:
            continue
        pattern = hist[L - n + 1:L + 1]
        ends = [e for e in range(L - 1, n - 2, -1) if hist[e - n + 1:e + 1] == pattern][:matches]
        for e in ends:
            cur = 0
            for tok in hist[e + 1:min(e + depth, L) + 1]:
                child = [t for t in range(1, len(ids)) if parents[t] == cur and ids[t] == tok]
                if not child and len(ids) == t_rows:
                    break
                if not child:
                    ids.append(tok)
                    parents.append(cur)
                    child = [len(ids) - 1]
                cur = child[0]
    pad = t_rows - len(ids)
    return ids + [0] * pad, parents + [-1] * pad


def ancestors(parents):
    """Per row the list of nodes from the root to the row itself, or None for
    a row that holds no node."""
    out = [[0]]
    for t in range(1, len(parents)):
        p = parents[t]
        out.append(out[p] + [t] if 0 <= p < t and out[p] is not None else None)
    return out


def accept(out_tok, ids, parents, hist, L, stop_len):
    """``(path, L')`` of one sequence; mutates ``hist``."""
    if L >= stop_len:
        return [], L
    path = [0]
    while True:
        cur = path[-1]
        child = [t for t in range(cur + 1, len(ids)) if parents[t] == cur and ids[t] == out_tok[cur]]
        if not child:
            break
        path.append(child[0])
    for i, t in enumerate(path):
        if 0 <= L + 1 + i < len(hist):
            hist[L + 1 + i] = out_tok[t]
    return path, L + len(path)


def bf(x):
    """Value of a float64 tensor after a round trip through bf16."""
    return x.to(torch.bfloat16).to(torch.float64)


def head_norm_rope(x, w, cos, sin, eps):
    """Per-head RMSNorm and RoPE of ``[..., D]`` rows, unrounded."""
    D = x.shape[-1]
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    rot = torch.cat((-y[..., D // 2:], y[..., :D // 2]), -1)
    return y * cos + rot * sin


def attention(qkv, parents, L, k_cache, v_cache, q_norm, k_norm, cos, sin, nq, nkv, eps, round_q=bf):
    """One sequence.  ``qkv`` [T, (nq + 2 nkv) D], ``k_cache`` / ``v_cache``
    [nkv, slots, D] (at least L slots), float64 throughout but for the queries
    (``round_q``) and node keys, which are rounded to bf16 once.  Returns ``out`` [T, nq, D],
    ``mag`` (the same sum over absolute values, the scale of its rounding
    errors), and the nodes' keys and values [nkv, T, D] (NaN in rows that hold
    no node)."""
    T, D = len(parents), cos.shape[-1]
    up = ancestors(parents)
    x = qkv.double().view(T, nq + 2 * nkv, D)
    out = torch.zeros((T, nq, D), dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    kn = torch.full((nkv, T, D), math.nan, dtype=torch.float64, device=x.device)
    vn = kn.clone()
    G = nq // nkv
    q = {}
    for t in range(T):
        if up[t] is None:
            continue
        pos = L + len(up[t]) - 1
        c, s = cos[pos].double(), sin[pos].double()
        q[t] = round_q(head_norm_rope(x[t, :nq], q_norm.double(), c, s, eps))
        kn[:, t] = bf(head_norm_rope(x[t, nq:nq + nkv], k_norm.double(), c, s, eps))
        vn[:, t] = x[t, nq + nkv:]
    kc, vc = k_cache[:, :L].double(), v_cache[:, :L].double()
    for t in q:
        keys, vals = torch.cat((kc, kn[:, up[t]]), 1), torch.cat((vc, vn[:, up[t]]), 1)
        p = torch.softmax(torch.matmul(q[t].view(nkv, G, D), keys.transpose(1, 2).contiguous()) / math.sqrt(D), -1)
        out[t] = torch.matmul(p, vals).view(nq, D)
        mag[t] = torch.matmul(p, vals.abs()).view(nq, D)
    return out, mag, kn, vn


def speculative_greedy(next_token, prompt, n_new, t_rows=8, primary=3, backoff=2, depth=4, matches=4):
    """Tree-speculative decoding of one sequence around ``next_token(prefix)``.
    Returns ``(tokens, iterations)``."""
    S = len(prompt)
    hist = list(prompt) + [0] * (n_new + t_rows + 1)
    hist[S] = next_token(list(prompt))
    L, stop, iters = S, S + n_new - 1, 0
    while L < stop:
        ids, parents = draft(hist, L, t_rows, primary, backoff, depth, matches)
        up = ancestors(parents)
        picks = [next_token(hist[:L] + [ids[j] for j in u]) if u else -1 for u in up]
        _, L = accept(picks, ids, parents, hist, L, stop)
        iters += 1
    return hist[S:S + n_new], iters
