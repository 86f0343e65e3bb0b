"""Tree speculation on top of ``DecodeState``: one pass verifies several
continuations of every sequence.

One iteration, captured as one hipGraph and replayed:

1. ``qdec_tree_draft``: what followed the ``matches`` most recent earlier
   occurrences of the last ``primary`` tokens, then of the last ``backoff``
   tokens, merged into a tree of at most ``nodes`` rows; the root is the
   current token.
2. one forward over ``nodes`` rows per sequence whose attention is
   ``qdec_tree_attn``: node t at position ``lens[b]`` + depth(t) sees the cache
   and its ancestors.  Node keys and values go to ``k_nodes`` / ``v_nodes``.
3. ``qdec_tree_accept``: the walk from the root along the greedy picks; its
   tokens are genuine greedy tokens and are appended to the history.
4. ``qdec_tree_commit``: the walk's keys and values into the cache, in every
   layer.  Nothing of the other branches ever reaches it.

Where a chain (``qdec.spec``) has one guess per position and none after its
first miss, the tree holds the alternatives that the history knows.  It costs
more rows: ``nodes`` is what TREE_ROWS leaves to a sequence.

Tokens.  Every emitted token is the greedy pick of its row.  The tree pass
rounds a node's key once where the plain step rounds it where the reference
does, and its attention sums in its own order, so at a near-tie the pick may
differ from the plain step's, as between two batch sizes of most engines; the
chain of ``qdec.spec`` is the mode that reproduces the plain stream bit for
bit.  Which kind of iteration runs follows from the tokens and the shape
(``tree_cost``), never from a clock: the same call gives the same tokens every time.

The acceptance gate is ``qdec.spec``'s: the drafter's rule restated on the host
(``TreeIndex``) scores every position with what a tree pass there would have
emitted, and tree passes run while that beats their cost; otherwise a plain step
keeps the history.
"""

import bisect

import torch

from . import capi
from .runtime import GEMM_MAX_ROWS, max_tree_nodes
from .spec import AcceptancePredictor, NgramIndex, SpecDecoder

# Rows of a tree pass, all sequences together.  Qwen3-4B's size, 1024 cached
# slots, batch 1 / 4 / 8, ms per iteration: plain 2.15 / 2.31 / 2.51, 16 rows 2.75 /
# 2.83 / 2.95, 32 rows 3.07 / 3.21 / 3.23, 48 rows 3.50 / 3.63 / 3.76, 64 rows 3.91 /
# 4.03 / 4.14: the second 16 rows cost 12%, the next ones 14% and 11%.
TREE_ROWS = 32
TREE_DEPTH = 8      # tokens taken from one earlier occurrence
TREE_MATCHES = 8    # earlier occurrences per pattern
# What a row past the plain step's adds to an iteration, in plain steps.
TREE_ROW_COST = 0.0135


def tree_cost(batch, nodes):
    """Plain steps that a tree pass of ``nodes`` rows per sequence costs: a part
    per row more, smaller where the plain step is itself of many rows.  A rule, not
    a time measured beside the run: the gate compares with it, and with a measured
    time the tokens at a near-tie would follow the clock.

    MI355X, rule / measured at 100, 1024 and 8192 cached slots.  Qwen3-4B's size,
    32 rows: batch 1 1.41 / 1.40 1.41 1.44, 2 1.39 / 1.34 1.36 1.25, 4 1.35 / 1.31
    1.38 1.28, 8 1.28 / 1.24 1.28 1.16, 16 1.16 / 1.04 1.07 1.04; 64 rows at 1024
    slots: batch 1 1.84 / 1.82, 4 1.76 / 1.74, 8 1.66 / 1.65.  28 layers of hidden
    2048, 32 rows: batch 1 1.41 / 1.42 1.32 1.32, 4 1.35 / 1.23 1.24 1.22."""
    return 1.0 + TREE_ROW_COST * batch * (nodes - 1) * (1.0 - batch / GEMM_MAX_ROWS)


def tree_nodes(batch):
    """Nodes per sequence, or 0 where TREE_ROWS leaves no room for a draft."""
    n = min(TREE_ROWS // batch, max_tree_nodes(batch))
    return n if n > 1 else 0


class TreeIndex(NgramIndex):
    """``draft(L)`` is the tree qdec_tree_draft makes at length L, as nested
    dicts from a token to its node's children."""

    def __init__(self, primary, backoff, depth, nodes, matches):
        super().__init__(primary, backoff, depth)
        self.nodes, self.matches = nodes, matches

    def draft(self, L):
        h, root, used = self.hist, {}, 1
        for n in self.ns:
            if L < n:
                continue
            found = self.starts[n].get(tuple(h[L - n + 1:L + 1]), ())
            i = bisect.bisect_left(found, L - n + 1)  # occurrences that end before L
            for j in reversed(found[max(0, i - self.matches):i]):
                cur = root
                for tok in h[j + n:min(j + n - 1 + self.k, L) + 1]:
                    if tok not in cur:
                        if used == self.nodes:
                            break
                        cur[tok] = {}
                        used += 1
                    cur = cur[tok]
        return root


class TreePredictor(AcceptancePredictor):
    """``AcceptancePredictor`` for trees: a position's sample is 1 + the steps
    of the walk along the greedy tokens that followed it."""

    def __init__(self, batch, primary, backoff, depth, nodes, matches):
        super().__init__(batch, primary, backoff, depth)
        self.index = [TreeIndex(primary, backoff, depth, nodes, matches) for _ in range(batch)]

    def _accepted(self, d, follow):
        a = 0
        while a < len(follow) and follow[a] in d:
            d = d[follow[a]]
            a += 1
        return a


class TreeDecoder(SpecDecoder):
    """``SpecDecoder``'s loop over tree iterations (``k`` = depth) and plain
    ones (``k`` = 0)."""

    def __init__(self, engine, state, primary, backoff, depth=TREE_DEPTH, matches=TREE_MATCHES):
        if state.tree_t < 2:
            raise ValueError(f"tree speculation needs a state with tree_t >= 2 (got {state.tree_t})")
        self.matches = matches
        super().__init__(engine, state, primary, backoff, depth)
        self.cost_ratio = tree_cost(state.batch, state.tree_t)

    def _buffers(self):
        st, dev = self.state, self.state.model.device
        self.T = st.tree_t
        self.naccept = st.naccept
        self.tokens = torch.zeros((st.batch * self.T,), dtype=torch.int64, device=dev)

    def _predictor(self):
        return TreePredictor(self.state.batch, self.primary, self.backoff, self.k, self.T, self.matches)

    def _rows(self, k):
        return self.T if k else 1

    def _checked(self, toks):
        self.engine._checked([t for t in toks if t != -1])  # -1: past a sequence's walk
        return toks

    def _stream(self):
        return torch.cuda.current_stream(self.state.model.device).cuda_stream

    def _draft(self, k):
        """The tree's ``ids`` and ``parents`` (k = 0: the current token)."""
        st = self.state
        self.lib.tree_draft(capi.TreeDraftArgs(
            hist=self.hist.data_ptr(), lens=st.lens.data_ptr(), ids=st.ids.data_ptr(), parents=st.parents.data_ptr(),
            batch=st.batch, cap=st.cap, t_rows=self._rows(k), primary=self.primary, backoff=self.backoff,
            depth=self.k, matches=self.matches), self._stream())

    def _iteration(self, k, stop_len):
        st = self.state
        self._draft(k)
        st.step(t_rows=self._rows(k), lm_head=True, ids_out=st.out_tok, advance=False, tree=k > 0)
        self.lib.tree_accept(capi.TreeAcceptArgs(
            out_tok=st.out_tok.data_ptr(), ids=st.ids.data_ptr(), parents=st.parents.data_ptr(),
            hist=self.hist.data_ptr(), lens=st.lens.data_ptr(), lens_out=st.lens.data_ptr(),
            naccept=self.naccept.data_ptr(), path=st.path.data_ptr(), emit=self.tokens.data_ptr(), batch=st.batch,
            cap=st.cap, t_rows=self._rows(k), stop_len=stop_len), self._stream())
        if k:  # a plain step wrote the cache itself
            st.tree_commit()
