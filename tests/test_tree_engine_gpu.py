"""Tree speculation through the engine: drafter, forward, acceptance and commit
together, as ``Engine(speculate="tree")`` runs them, against the model's oracle
and the plain path.

A tree pass rounds keys and sums differently from the plain step, so tokens are
judged as the other head layouts' are (tests/test_shapes_gpu.py): every token
is the oracle's argmax after the engine's own prefix, or the oracle's top-2 gap
there is below 2e-2 of the row's largest |logit|.  Against the plain tokens
every difference has to begin at such a near-tie."""

import pytest
import torch

from oracle.qwen3_oracle import Qwen3Oracle, top2_gap
from qdec.checkpoint import load_tensors, qwen3_config, write_checkpoint

pytestmark = pytest.mark.gpu

TOL = 2e-2

SHAPES = {
    "g2": dict(hidden_size=2048, intermediate_size=6144, num_attention_heads=16, num_key_value_heads=8),
    "g4": {},
    "tiny": dict(hidden_size=256, intermediate_size=768, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                 vocab_size=1024, tie_word_embeddings=True),
}


@pytest.fixture(scope="module", params=sorted(SHAPES))
def model(request, tmp_path_factory):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    from engine import Engine
    cfg = qwen3_config(num_hidden_layers=2, **SHAPES[request.param])
    path = str(tmp_path_factory.mktemp(f"qwen3_tree_{request.param}"))
    write_checkpoint(path, cfg, seed=5, norm_jitter=0.05)
    eng = Engine(path, speculate="tree")
    ora = Qwen3Oracle(cfg, load_tensors(path), mode="bf16", attn="decode")
    yield request.param, cfg, eng, ora
    del eng
    torch.cuda.empty_cache()


def motif_prompts(vocab, B, S, seed, motif=12, noise=0.15):
    g = torch.Generator().manual_seed(seed)
    base = torch.randint(0, vocab, (motif,), generator=g)
    rows = []
    for _ in range(B):
        r = base.repeat((S + motif - 1) // motif)[:S].clone()
        m = torch.rand(S, generator=g) < noise
        r[m] = torch.randint(0, vocab, (int(m.sum()),), generator=g)
        rows.append(r)
    return torch.stack(rows)


def judge(ora, prompt, steps):
    toks = torch.tensor(steps).T.contiguous()  # [B, n]
    ref = ora.teacher_forced(prompt, toks)
    miss = ref.argmax(-1) != toks
    near = top2_gap(ref) < TOL * ref.abs().amax(-1)
    assert bool((~miss | near).all()), f"non-near-tie divergence: {miss.nonzero().tolist()}"
    return near


def check_prefix(near, got, plain):
    """Rows of ``got`` equal ``plain`` up to a near-tie."""
    got, plain = torch.tensor(got).T, torch.tensor(plain).T
    for b in range(got.shape[0]):
        d = (got[b] != plain[b]).nonzero()
        assert len(d) == 0 or bool(near[b, int(d[0])]), (b, int(d[0]))


@pytest.mark.parametrize("B,S,n", [(1, 60, 24), (1, 300, 10), (4, 100, 16), (16, 30, 8), (40, 17, 4), (2, 5, 1)])
def test_engine_tree_tokens(model, B, S, n):
    """Both with every pass a tree and under the gate; 40 sequences leave no
    room for a tree and run plain steps; one token needs no pass at all."""
    name, cfg, eng, ora = model
    prompt = motif_prompts(cfg["vocab_size"], B, S, 31 + B + S)
    eng.speculate = False
    plain = list(eng.generate(prompt.tolist(), n))
    eng.speculate = "tree"
    for gate in (False, True):
        eng.spec_gate = gate
        steps = list(eng.generate(prompt.tolist(), n))
        stats = eng.stats["spec"]
        print(f"{name} B={B} S={S} gate={gate}: {stats}", flush=True)
        check_prefix(judge(ora, prompt, steps), steps, plain)
        assert len(steps) == n and stats["iterations"] <= n - 1
        if B > 16:
            assert steps == plain and stats["verify_iterations"] == 0
        elif not gate:
            assert stats["plain_iterations"] == 0
            assert list(eng.generate(prompt.tolist(), n)) == steps  # the graphs replay to the same tokens


def planted(dec, plain, S, width):
    """A ``_draft`` whose trees hold the plain run's next tokens under
    ``width`` wrong siblings each: B host-built trees per pass."""
    st, T = dec.state, dec.T

    def draft(k):
        assert k > 0
        ids, parents = [], []
        for b, L in enumerate(st.lens.tolist()):
            t_ids, t_par, cur = [int(dec.hist[b, L])], [-1], 0
            for tok in [s[b] for s in plain[L - S + 1:]]:
                if len(t_ids) + width >= T:
                    break
                for w in range(width):
                    t_ids.append((tok + 1 + w) % 1000)
                    t_par.append(cur)
                t_ids.append(tok)
                t_par.append(cur)
                cur = len(t_ids) - 1
            pad = T - len(t_ids)
            ids += t_ids + [0] * pad
            parents += t_par + [-1] * pad
        st.ids[:len(ids)].copy_(torch.tensor(ids))
        st.parents.copy_(torch.tensor(parents, dtype=torch.int32))

    return draft


@pytest.mark.parametrize("B,S,n,width", [(1, 40, 40, 1), (3, 90, 24, 2), (8, 33, 12, 0)])
def test_long_walks(model, B, S, n, width):
    """Trees that hold the right continuation among wrong siblings: walks of
    several nodes, whose keys and values later passes read from the cache."""
    from qdec.runtime import DecodeState
    from qdec.tree import TreeDecoder, tree_nodes
    name, cfg, eng, ora = model
    prompt = motif_prompts(cfg["vocab_size"], B, S, 77 + B)
    eng.speculate = False
    plain = list(eng.generate(prompt.tolist(), n))
    T = tree_nodes(B)
    st = DecodeState(eng.model, B, S + n + 2 * T, max_t=16, tree_t=T)
    graphs, eng.use_graphs = eng.use_graphs, False
    try:
        dec = TreeDecoder(eng, st, 3, 2)
        dec._draft = planted(dec, plain, S, width)
        steps = list(dec.generate(prompt, n, gate=False))
    finally:
        eng.use_graphs = graphs
    check_prefix(judge(ora, prompt, steps), steps, plain)
    print(f"{name} B={B}: {dec.last_stats['iterations']} passes for {n} tokens", flush=True)
    if steps == plain:  # every planted walk was accepted whole
        per = (T - 1) // (width + 1) + 1
        assert dec.last_stats["iterations"] <= -(-(n - 1) // per) + 1


@pytest.mark.parametrize("B", [1, 3, 16, 32])
def test_widest_trees(model, B):
    """States of as many nodes as the GEMMs take: the known-answer checks, and
    planted walks."""
    from qdec import selfcheck
    from qdec.runtime import DecodeState, max_tree_nodes
    from qdec.tree import TreeDecoder
    name, cfg, eng, ora = model
    S, n, T = 24, 10, max_tree_nodes(B)
    prompt = motif_prompts(cfg["vocab_size"], B, S, 55 + B)
    eng.speculate = False
    plain = list(eng.generate(prompt.tolist(), n))
    st = DecodeState(eng.model, B, S + n + 2 * T, max_t=16, tree_t=T)
    selfcheck.run_tree(st)
    graphs, eng.use_graphs = eng.use_graphs, False
    try:
        dec = TreeDecoder(eng, st, 3, 2)
        dec._draft = planted(dec, plain, S, 1 if T > 2 else 0)
        steps = list(dec.generate(prompt, n, gate=False))
    finally:
        eng.use_graphs = graphs
    check_prefix(judge(ora, prompt, steps), steps, plain)


def test_iteration_captured_and_replayed(model):
    """One whole iteration as a graph, replayed with other work between,
    against eager iterations from the same start: every buffer bit for bit."""
    from qdec.runtime import DecodeState
    from qdec.tree import TreeDecoder, tree_nodes
    name, cfg, eng, _ = model
    B, S, n = 3, 70, 40
    T = tree_nodes(B)
    prompt = motif_prompts(cfg["vocab_size"], B, S, 5).to(eng.device)
    runs = []
    for captured in (False, True):
        st = DecodeState(eng.model, B, S + n + 2 * T, max_t=16, tree_t=T)
        dec = TreeDecoder(eng, st, 2, 1)
        if captured:
            graph = eng._capture(lambda: dec._iteration(dec.k, S + n))
        st.prefill(prompt)
        dec.hist.zero_()
        dec.hist[:, :S].copy_(prompt)
        dec.hist[:, S].copy_(st.ids[:B])
        seen = []
        for _ in range(5):
            graph.replay() if captured else dec._iteration(dec.k, S + n)
            seen.append([t.clone() for t in (st.lens, dec.hist, dec.tokens, st.path, st.naccept, st.parents)])
            torch.randn(512, 512, device=eng.device).sum().item()
        cut = int(st.lens.min())
        seen.append([st.k_cache[:, :, :, :cut].clone(), st.v_cache[:, :, :, :cut // 8 * 8].clone()])
        runs.append(seen)
    for i, (x, y) in enumerate(zip(*runs)):
        for j, (p, q) in enumerate(zip(x, y)):
            assert torch.equal(p, q), (name, i, j)


def test_refusals(model):
    from qdec.runtime import DecodeState, max_tree_nodes
    from qdec.tree import TreeDecoder
    _, _, eng, _ = model
    with pytest.raises(ValueError, match="tree_t"):
        DecodeState(eng.model, 4, 64, max_t=1, tree_t=max_tree_nodes(4) + 1)
    st = DecodeState(eng.model, 2, 64, max_t=1)
    with pytest.raises(ValueError, match="tree_t"):
        st.run_step(t_rows=4, advance=False, tree=True)
    with pytest.raises(ValueError, match="tree_t"):
        TreeDecoder(eng, st, 3, 2)
    st = DecodeState(eng.model, 2, 64, max_t=1, tree_t=4)
    with pytest.raises(ValueError, match="tree_t"):
        st.run_step(t_rows=3, advance=False, tree=True)
    with pytest.raises(ValueError, match="advance"):
        st.run_step(t_rows=4, tree=True)
    with pytest.raises(ValueError, match="t_rows"):
        st.run_step(t_rows=4, advance=False)
    dec = TreeDecoder(eng, st, 3, 2)
    with pytest.raises(ValueError, match="capacity"):
        next(dec.generate(torch.zeros((2, 40), dtype=torch.int64), 30))
