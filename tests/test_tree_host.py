"""The host side of tree speculation, without a GPU: the index the acceptance
gate uses restates the device drafter, and the predictor scores every position
with the walk a tree pass there would have made."""

import random

import pytest

from oracle import tree_oracle
from qdec.tree import TREE_DEPTH, TREE_MATCHES, TreeIndex, TreePredictor, tree_nodes


def as_dict(ids, parents):
    """The oracle's tree as nested dicts."""
    nodes = [{}]
    for t in range(1, len(ids)):
        if parents[t] < 0:
            break
        nodes.append({})
        nodes[parents[t]][ids[t]] = nodes[t]
    return nodes[0]


def test_index_equals_drafter_on_random_histories():
    rng = random.Random(0)
    for _ in range(300):
        n, alphabet = rng.randint(1, 70), rng.choice([1, 2, 4, 30])
        hist = [rng.randrange(alphabet) for _ in range(n)]
        T, depth, matches = rng.randint(2, 20), rng.randint(1, 9), rng.randint(1, 5)
        primary, backoff = rng.randint(1, 4), rng.randint(1, 4)
        ix = TreeIndex(primary, backoff, depth, T, matches)
        for L, t in enumerate(hist):
            ix.append(t)
            ids, parents = tree_oracle.draft(hist + [0] * 9, L, T, primary, backoff, depth, matches)
            assert ix.draft(L) == as_dict(ids, parents), (hist, L)


def test_predictor_scores_what_a_tree_pass_would_accept():
    rng = random.Random(1)
    for _ in range(60):
        T, depth, matches = rng.randint(2, 12), rng.randint(1, 6), rng.randint(1, 4)
        prompt = [rng.randint(0, 3) for _ in range(rng.randint(1, 20))]
        gen = [rng.randint(0, 3) for _ in range(rng.randint(depth + 1, 40))]
        p = TreePredictor(1, 3, 2, depth, T, matches)
        p.start(0, prompt, gen[0])
        for i in range(1, len(gen), 3):
            p.extend(0, gen[i:i + 3])
        hist, want = prompt + gen, []
        for L in range(len(prompt), len(hist) - depth):
            ids, parents = tree_oracle.draft(hist + [0] * 9, L, T, 3, 2, depth, matches)
            up = tree_oracle.ancestors(parents)
            picks = [hist[L + len(u)] if u and L + len(u) < len(hist) else -1 for u in up]
            path, _ = tree_oracle.accept(picks, ids, parents, list(hist) + [0] * 20, L, 10 ** 9)
            want.append(len(path))
        assert (p.positions, p.total, p.hits) == (len(want), sum(want), sum(w > 1 for w in want))


@pytest.mark.parametrize("batch", range(1, 65))
def test_nodes_per_sequence(batch):
    """Within the drafter's and the attention's limits and the GEMMs' rows."""
    from qdec import capi
    from qdec.runtime import GEMM_MAX_ROWS, max_tree_nodes
    n = tree_nodes(batch)
    assert n == 0 or 2 <= n <= min(max_tree_nodes(batch), capi.TREE_MAX_T) and batch * n <= GEMM_MAX_ROWS
    assert 1 <= TREE_DEPTH < capi.TREE_MAX_T and 1 <= TREE_MATCHES <= capi.TREE_MAX_MATCHES


def test_engine_speculation_modes():
    from engine import speculation
    assert [speculation(m) for m in (False, True, None, 1, "tree")] == [False, True, False, True, "tree"]
    with pytest.raises(ValueError, match="speculate"):
        speculation("chain")
