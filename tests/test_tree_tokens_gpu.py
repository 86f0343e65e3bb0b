"""Tokens of ``Engine(speculate="tree")``, judged by the token that was emitted:
its own logit in the oracle, after the engine's own prefix, is within 2e-2 of the
row's largest |logit| of the largest one.  And walks of known length: trees that
hold the run's own continuation are accepted whole."""

import pytest
import torch
from test_tree_engine_gpu import TOL, model, motif_prompts, planted  # noqa: F401  (model: the fixture)

pytestmark = pytest.mark.gpu


def judge_tokens(ora, prompt, steps):
    toks = torch.tensor(steps).T.contiguous()  # [B, n]
    ref = ora.teacher_forced(prompt, toks)
    own = ref.gather(-1, toks[..., None])[..., 0]
    short = (ref.amax(-1) - own) / ref.abs().amax(-1)
    assert bool((short <= TOL).all()), (short > TOL).nonzero().tolist()


@pytest.mark.parametrize("B,S,n", [(1, 60, 24), (2, 200, 12), (4, 100, 16), (16, 30, 8)])
def test_every_token_is_a_greedy_one(model, B, S, n):  # noqa: F811
    name, cfg, eng, ora = model
    prompt = motif_prompts(cfg["vocab_size"], B, S, 131 + B + S)
    eng.speculate = "tree"
    for gate in (False, True):
        eng.spec_gate = gate
        judge_tokens(ora, prompt, list(eng.generate(prompt.tolist(), n)))


@pytest.mark.parametrize("B,S,n,width", [(1, 40, 40, 1), (3, 90, 24, 2), (8, 33, 12, 0)])
def test_planted_walks_are_accepted_whole(model, B, S, n, width):  # noqa: F811
    """The trees hold the tokens of the run before; where a near-tie turned one,
    the next run plants the new stream.  A node's row does not depend on the other
    branches, so what came before that token stays, and the streams settle."""
    from qdec.runtime import DecodeState
    from qdec.tree import TreeDecoder, tree_nodes
    name, cfg, eng, ora = model
    prompt = motif_prompts(cfg["vocab_size"], B, S, 177 + B)
    eng.speculate = False
    steps = list(eng.generate(prompt.tolist(), n))
    T = tree_nodes(B)
    st = DecodeState(eng.model, B, S + n + 2 * T, max_t=16, tree_t=T)
    graphs, eng.use_graphs = eng.use_graphs, False
    try:
        dec = TreeDecoder(eng, st, 3, 2)
        for run in range(n):
            dec._draft = planted(dec, steps, S, width)
            before, steps = steps, list(dec.generate(prompt, n, gate=False))
            if steps == before:
                break
    finally:
        eng.use_graphs = graphs
    assert steps == before, run
    judge_tokens(ora, prompt, steps)
    per = (T - 1) // (width + 1) + 1
    print(f"{name} B={B}: settled after {run + 1} runs, {dec.last_stats['iterations']} passes for {n} tokens", flush=True)
    assert dec.last_stats["iterations"] == -(-(n - 1) // per)


@pytest.mark.parametrize("B,S,n", [(1, 60, 64), (4, 50, 48)])
def test_gated_runs_repeat(model, monkeypatch, B, S, n):  # noqa: F811
    """In graphs, again, and eagerly: the same tokens from the same iterations,
    with the rule's cost and with one that any accepted draft outweighs."""
    from qdec import tree
    name, cfg, eng, ora = model
    prompt = motif_prompts(cfg["vocab_size"], B, S, 11 + B)
    eng.speculate, eng.spec_gate, graphs = "tree", True, eng.use_graphs
    try:
        for cost in (tree.tree_cost, lambda batch, nodes: 0.96):
            monkeypatch.setattr(tree, "tree_cost", cost)
            seen = []
            for use in (True, True, False):
                eng.use_graphs, eng.shape = use, None
                steps = list(eng.generate(prompt.tolist(), n))
                seen.append((steps, {k: eng.stats["spec"][k] for k in ("iterations", "verify_iterations", "cost_ratio")}))
            print(f"{name} B={B}: {seen[0][1]}", flush=True)
            assert seen[0] == seen[1] == seen[2]
    finally:
        eng.use_graphs, eng.shape = graphs, None
