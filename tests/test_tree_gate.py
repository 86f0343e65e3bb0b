"""The gate of tree speculation decides by rules, not by a clock: with it, too,
the same call gives the same tokens every time, in graphs as in eager runs."""

import types

import pytest
import torch

from qdec import spec, tree


def decoder(batch, nodes, use_graphs, monkeypatch, ms):
    """A TreeDecoder on a state of host tensors whose graphs record nothing;
    `ms` is what a clock would say of the tree's and the plain iteration."""
    st = types.SimpleNamespace(batch=batch, cap=256, tree_t=nodes, lib=None, lens=torch.zeros(batch, dtype=torch.int32),
                               naccept=torch.zeros(batch, dtype=torch.int32),
                               model=types.SimpleNamespace(device=torch.device("cpu")))
    times = iter(ms)

    class Event:
        def __init__(self, **kw):
            pass

        def record(self):
            pass

        def elapsed_time(self, other):
            return next(times)

    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    eng = types.SimpleNamespace(use_graphs=use_graphs, _capture=lambda fn: types.SimpleNamespace(replay=lambda: None))
    dec = tree.TreeDecoder(eng, st, 3, 2)
    dec._ensure_graphs(100)
    return dec


@pytest.mark.parametrize("batch,nodes", [(1, 32), (4, 8), (16, 2), (1, 64), (32, 2)])
def test_cost_does_not_come_from_a_clock(monkeypatch, batch, nodes):
    seen = {decoder(batch, nodes, graphs, monkeypatch, ms).cost_ratio
            for graphs, ms in ((True, (1.0, 5.0)), (True, (5.0, 1.0)), (False, (1.0, 1.0)))}
    assert len(seen) == 1 and None not in seen
    ratio = seen.pop()
    # dearer than a plain step, and the margin leaves the gate something a full tree can reach
    assert 1.0 < ratio and ratio * spec.MARGIN < min(nodes, tree.TREE_DEPTH + 1)


def test_cost_grows_with_the_rows():
    for batch in (1, 2, 4, 8, 16):
        costs = [tree.tree_cost(batch, n) for n in range(1, 64 // batch + 1)]
        assert costs[0] == 1.0 and costs == sorted(costs)
