"""The restatement of tree speculation, pinned by known answers, brute force,
the chain rules it contains and the tree == plain greedy invariant."""

import random

import torch

from oracle import spec_oracle, tree_oracle


def test_draft_known_answers():
    #        0  1  2  3  4  5  6  7  8  9 10 11 12 13
    hist = [1, 2, 3, 7, 1, 2, 3, 8, 9, 5, 1, 2, 3, 0]
    # 1 2 3 ended at 6 (then 8 9 5) and at 2 (then 7 1 2)
    ids, par = tree_oracle.draft(hist, 12, 8, 3, 2, 3, 4)
    assert ids == [3, 8, 9, 5, 7, 1, 2, 0] and par == [-1, 0, 1, 2, 0, 4, 5, -1]
    # the budget ends inside the second candidate
    assert tree_oracle.draft(hist, 12, 5, 3, 2, 3, 4) == ([3, 8, 9, 5, 7], [-1, 0, 1, 2, 0])
    # one candidate per pattern: 2 3 finds the same place again
    assert tree_oracle.draft(hist, 12, 8, 3, 2, 2, 1) == ([3, 8, 9, 0, 0, 0, 0, 0], [-1, 0, 1] + [-1] * 5)
    # nothing repeats; too short for any pattern; one row
    assert tree_oracle.draft([1, 2, 3, 4], 3, 3, 3, 2, 2, 2) == ([4, 0, 0], [-1, -1, -1])
    assert tree_oracle.draft([9, 0], 0, 2, 3, 2, 2, 2) == ([9, 0], [-1, -1])
    assert tree_oracle.draft(hist, 12, 1, 3, 2, 3, 4) == ([3], [-1])
    # a run of one token: its occurrences merge into one chain, cut at the history's end
    assert tree_oracle.draft([4] * 6, 5, 8, 2, 1, 3, 8) == ([4, 4, 4, 4, 0, 0, 0, 0], [-1, 0, 1, 2] + [-1] * 4)


def test_draft_first_branch_is_the_most_recent_match():
    rng = random.Random(3)
    for _ in range(200):
        hist = [rng.randint(0, 3) for _ in range(rng.randint(4, 40))]
        L = rng.randint(3, len(hist) - 1)
        ids, par = tree_oracle.draft(hist, L, 16, 3, 2, 4, 6)
        for t in range(1, 16):  # a parent precedes its children, siblings differ
            assert par[t] < t
            if par[t] < 0:
                assert ids[t:] == [0] * (16 - t) and par[t:] == [-1] * (16 - t)
                break
            assert all(ids[u] != ids[t] for u in range(1, t) if par[u] == par[t])
        ends = [e for e in range(2, L) if hist[e - 2:e + 1] == hist[L - 2:L + 1]]
        if ends:
            first = hist[ends[-1] + 1:min(ends[-1] + 4, L) + 1]
            assert ids[1:1 + len(first)] == first and par[1:1 + len(first)] == list(range(len(first)))


def test_ancestors_and_accept():
    par = [-1, 0, 1, 0, 3, 9, 5, 4, -1, 8]
    up = tree_oracle.ancestors(par)
    assert up[2] == [0, 1, 2] and up[4] == [0, 3, 4] and up[7] == [0, 3, 4, 7]
    assert up[5] is None and up[6] is None and up[8] is None and up[9] is None
    ids = [10, 11, 12, 13, 14, 13, 0, 15, 0, 0]
    hist = [1, 2, 3, 10, 0, 0, 0, 0]
    picks = [13, 0, 0, 14, 15, 0, 0, 77, 0, 0]
    assert tree_oracle.accept(picks, ids, par, hist, 3, 100) == ([0, 3, 4, 7], 7)
    assert hist == [1, 2, 3, 10, 13, 14, 15, 77]
    assert tree_oracle.accept(picks, ids, par, hist, 7, 7) == ([], 7)


def test_a_chain_is_the_chain_rule():
    rng = random.Random(5)
    for _ in range(200):
        k = rng.randint(1, 6)
        d = [rng.randint(0, 2) for _ in range(k)]
        picks = [rng.randint(0, 2) for _ in range(k + 1)]
        hist = [rng.randint(0, 2) for _ in range(12)]
        L = rng.randint(0, 11)
        h1, h2 = list(hist), list(hist)
        a, L1 = spec_oracle.accept(picks, d, h1, L, k, 11)
        path, L2 = tree_oracle.accept(picks, [hist[L]] + d, list(range(-1, k)), h2, L, 11)
        assert (len(path) - 1 if path else 0, h1, L1) == (a, h2, L2)


def test_tree_speculation_equals_plain_greedy():
    rng = random.Random(11)
    for trial in range(20):
        table = [rng.randint(0, 5) for _ in range(36)]

        def nxt(prefix):
            return table[(prefix[-1] * 6 + (prefix[-2] if len(prefix) > 1 else 0)) % 36]

        prompt = [rng.randint(0, 5) for _ in range(rng.randint(1, 12))]
        n = rng.randint(1, 40)
        plain = spec_oracle.plain_greedy(nxt, prompt, n)
        toks, iters = tree_oracle.speculative_greedy(nxt, prompt, n, t_rows=rng.randint(1, 9))
        assert toks == plain and iters <= max(n - 1, 0)


def test_attention_of_a_chain_is_causal_attention():
    g = torch.Generator().manual_seed(0)
    T, L, nq, nkv, D = 5, 7, 4, 2, 8
    qkv = torch.randn(T, (nq + 2 * nkv) * D, generator=g).double()
    kc, vc = (torch.randn(nkv, L, D, generator=g).double() for _ in range(2))
    one = torch.ones(D)
    ang = torch.randn(16, D // 2, generator=g)
    cos, sin = torch.cat((ang.cos(),) * 2, 1), torch.cat((ang.sin(),) * 2, 1)
    out, mag, kn, vn = tree_oracle.attention(qkv, [-1, 0, 1, 2, 3], L, kc, vc, one, one, cos, sin, nq, nkv, 1e-6)
    x = qkv.view(T, nq + 2 * nkv, D)
    q = torch.stack([tree_oracle.bf(tree_oracle.head_norm_rope(x[t, :nq], one.double(), cos[L + t].double(),
                                                               sin[L + t].double(), 1e-6)) for t in range(T)], 1)
    keys, vals = torch.cat((kc, kn), 1).repeat_interleave(2, 0), torch.cat((vc, vn), 1).repeat_interleave(2, 0)
    s = q @ keys.transpose(1, 2).contiguous() / D ** 0.5
    s = s.masked_fill(torch.arange(L + T)[None] > L + torch.arange(T)[:, None], -torch.inf)
    ref = (s.softmax(-1) @ vals).transpose(0, 1)
    assert (out - ref).abs().max() < 1e-12 and (mag >= out.abs() - 1e-12).all()
    assert torch.equal(vn, x[:, nq + nkv:].transpose(0, 1))
