"""The engine with an 8-bit KV cache (``Engine(kv_cache="int8")``) end to end:
prompts, steps, graphs and speculation over it.

The oracle holds the key and value rows it writes as the cache does
(oracle/kv8_oracle.py).  A key near a rounding border may fall to the other
side in one of the two, since the prompt kernels round keys to bf16 before they
are held and the steps do not; so logits are judged as elsewhere, within 2e-2 of the row's
largest |logit|, and tokens by the oracle's argmax or a top-2 gap below that."""

import pytest
import torch

from oracle import kv8_oracle
from oracle.qwen3_oracle import Qwen3Oracle, normalized_max_err, top2_gap
from qdec.checkpoint import load_tensors, qwen3_config, write_checkpoint

pytestmark = pytest.mark.gpu

TOL = 2e-2

SHAPES = {
    "g2": dict(hidden_size=2048, intermediate_size=6144, num_attention_heads=16, num_key_value_heads=8),
    "g4": {},
    "g5": dict(hidden_size=640, intermediate_size=1280, num_attention_heads=10, num_key_value_heads=2, vocab_size=2048),
    "tiny": dict(hidden_size=256, intermediate_size=768, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                 vocab_size=1024, tie_word_embeddings=True),
}


def held(rows):
    q, s = kv8_oracle.hold(rows)
    return (q * s.float().double()[..., None]).float()


@pytest.fixture(scope="module", params=sorted(SHAPES))
def model(request, tmp_path_factory):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    from engine import Engine
    cfg = qwen3_config(num_hidden_layers=2, **SHAPES[request.param])
    path = str(tmp_path_factory.mktemp(f"qwen3_kv8_{request.param}"))
    write_checkpoint(path, cfg, seed=5, norm_jitter=0.05)
    eng = Engine(path, kv_cache="int8")
    ora = Qwen3Oracle(cfg, load_tensors(path), mode="bf16", attn="decode", hold=held)
    yield request.param, cfg, eng, ora
    del eng
    torch.cuda.empty_cache()


def prompts(vocab, B, S, seed, motif=0):
    g = torch.Generator().manual_seed(seed)
    if not motif:
        return torch.randint(0, vocab, (B, S), generator=g)
    base = torch.randint(0, vocab, (B, motif), generator=g)
    return base.repeat(1, S // motif + 1)[:, :S]


def state(eng, B, cap, **kw):
    from qdec.runtime import DecodeState
    return DecodeState(eng.model, B, cap, max_t=16, kv8=True, **kw)


@pytest.mark.parametrize("B,S,n", [(1, 5, 6), (2, 40, 4), (3, 70, 4), (1, 300, 3), (12, 90, 3)])
def test_logits_and_tokens_vs_oracle(model, B, S, n):
    name, cfg, eng, ora = model
    prompt = prompts(cfg["vocab_size"], B, S, 7 * B + S)
    st = state(eng, B, S + n + 2, keep_logits=True)
    st.prefill(prompt.to(eng.device))
    toks, logits = [st.ids[:B].cpu()], [st.logits[:B].float().cpu()]
    for _ in range(n - 1):
        st.run_step(t_rows=1)
        toks.append(st.ids[:B].cpu())
        logits.append(st.logits[:B].float().cpu())
    toks, logits = torch.stack(toks, 1), torch.stack(logits, 1)
    ref = ora.teacher_forced(prompt, toks)
    err = normalized_max_err(logits, ref).max().item()
    print(f"{name} B={B} S={S}: normalised max err {err:.4g}")
    assert err <= TOL
    near = top2_gap(ref) < TOL * ref.abs().amax(-1)
    assert bool(((ref.argmax(-1) == toks) | near).all())
    assert list(eng.generate(prompt.tolist(), n)) == toks.T.tolist()  # the replayed graph


def test_speculation_gives_the_plain_tokens(model):
    name, cfg, eng, _ = model
    for B, S in ((1, 60), (2, 33), (4, 100)):
        prompt = prompts(cfg["vocab_size"], B, S, 3 + B, motif=9).tolist()
        eng.speculate = False
        plain = list(eng.generate(prompt, 40))
        eng.speculate, eng.spec_gate = True, False
        try:
            assert list(eng.generate(prompt, 40)) == plain, (name, B)
            assert eng.stats["spec"]["verify_iterations"] > 0 or B > 2
        finally:
            eng.speculate, eng.spec_gate = False, True


def test_prompt_in_chunks_is_the_same_prompt(model):
    """Later chunks read the earlier ones back from the cache: cache, picks and
    logits are bit for bit those of the whole prompt."""
    from qdec.runtime import Prefill
    name, cfg, eng, _ = model
    if not eng.model.cfg.prefill_kernels:
        pytest.skip("prompts of this head layout run through the decode kernels")
    for B, S, rows in ((1, 300, 70), (2, 130, 64), (3, 40, 51)):
        prompt = prompts(cfg["vocab_size"], B, S, 11 + S).to(eng.device)
        got = []
        for r in (None, rows):
            st = state(eng, B, S + 8, keep_logits=True)
            Prefill(st, S, **({"rows": r} if r else {})).run(prompt)
            st.run_step(t_rows=1)
            torch.cuda.synchronize()
            got.append([x.clone() for x in (st.k8, st.v8, st.k_scale, st.v_scale, st.ids, st.logits[:B])])
        for x, y in zip(*got):
            assert torch.equal(x, y), (name, B, S, rows)


def test_a_longer_prompt_after_a_shorter_one(model):
    """The slabs that prompts share grow with the prompt."""
    name, cfg, eng, _ = model
    long = prompts(cfg["vocab_size"], 2, 200, 21).to(eng.device)
    want = state(eng, 2, 264, keep_logits=True)
    want.prefill(long)
    st = state(eng, 2, 264, keep_logits=True)
    st.prefill(long[:, :50].contiguous())
    st.prefill(long)
    assert torch.equal(st.logits[:2], want.logits[:2]) and torch.equal(st.k8, want.k8)


@pytest.mark.parametrize("S", [500, 700, 1500])
def test_attention_merged_in_o(model, monkeypatch, S):
    """The steps whose O projection merges the attention's partials have the bits of
    those whose attention does, and so do verify passes."""
    name, cfg, eng, _ = model
    if eng.model.cfg.group != 4 or eng.model.cfg.head_dim != 128:
        pytest.skip("O merges 4 query heads of 128 channels per kv head")
    B = 1
    prompt = prompts(cfg["vocab_size"], B, S, S).to(eng.device)
    got = []
    for merge in (True, False):
        st = state(eng, B, 1700, keep_logits=True)
        assert st._merge_in_o(1) and not st._merge_in_o(2)
        if not merge:
            monkeypatch.setattr(st, "_merge_in_o", lambda t: False)
        st.prefill(prompt)
        rows = []
        for _ in range(3):
            st.run_step()
            rows.append((st.logits[:B].clone(), st.ids[:B].clone()))
        got.append(rows)
    for x, y in zip(*got):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    # one workgroup takes a sequence; many partials; two sequences
    assert not any(state(eng, b, cap)._merge_in_o(1) for b, cap in ((1, 500), (1, 4200), (2, 1700)))


def test_long_speculation_gives_the_plain_tokens(model):
    name, cfg, eng, _ = model
    for B, S in ((1, 1100), (2, 1030)):
        prompt = prompts(cfg["vocab_size"], B, S, 5 + B, motif=9).tolist()
        plain = list(eng.generate(prompt, 30))
        eng.speculate, eng.spec_gate = True, False
        try:
            assert list(eng.generate(prompt, 30)) == plain, (name, B)
        finally:
            eng.speculate, eng.spec_gate = False, True


def test_memory(model):
    _, _, eng, _ = model
    from qdec.runtime import DecodeState
    st, bf = state(eng, 2, 512), DecodeState(eng.model, 2, 512, max_t=16)
    held8 = sum(x.numel() * x.element_size() for x in (st.k8, st.v8, st.k_scale, st.v_scale))
    both = sum(x.numel() * x.element_size() for x in (bf.k_cache, bf.v_cache))
    assert held8 <= both * (0.5 + 2 / eng.model.cfg.head_dim)
    assert not hasattr(st, "k_cache")


def test_refusals(model, monkeypatch):
    from engine import Engine
    from qdec.runtime import DecodeState
    _, cfg, eng, _ = model
    with pytest.raises(ValueError, match="tree"):
        DecodeState(eng.model, 2, 64, tree_t=4, kv8=True)
    monkeypatch.setattr(eng, "speculate", "tree")
    with pytest.raises(ValueError, match="tree"):
        next(eng.generate([[1, 2, 3]], 4))
    monkeypatch.setattr(eng, "speculate", False)
    monkeypatch.setattr(eng, "kv_cache", "fp8")
    with pytest.raises(ValueError, match="kv_cache"):
        next(eng.generate([[1, 2, 3]], 4))
    st = state(eng, 2, 64)
    assert not st.layer_supported()
    with pytest.raises(ValueError, match="bf16"):
        st.enable_layer_launch()
