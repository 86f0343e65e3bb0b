"""What a result of the tree attention depends on: a row's bits follow from its
own query, what it sees, the splits, its sequence's length and the call's shape.
Neither the other sequences' lengths nor the other rows of its own sequence
move them."""

import pytest
import torch
from test_tree_gpu import DEV, Attn, i32, lib  # noqa: F401  (lib: the fixture)

from qdec import capi

pytestmark = pytest.mark.gpu


def group_rows(c, n):
    """The call's row groups are of n rows, as the partials' size shows."""
    a = capi.TreeAttnArgs.from_buffer_copy(c.a)
    a.splits = 2
    groups = -(-c.T * (c.nq // c.nkv) // n)
    return c.lib.tree_attn_workspace(a)[0] == 4 * c.B * c.nkv * 2 * groups * n * (c.D + 2)


def bits(*tensors):
    return [t.clone().view(torch.int16) for t in tensors]


# T, query heads, kv heads, head_dim, cap, splits, rows of a group
NEIGHBOURS = [(8, 32, 8, 128, 1088, 0, 32), (8, 32, 8, 128, 1088, 4, 32), (3, 8, 2, 128, 1088, 4, 16),
              (40, 8, 2, 64, 2080, 3, 32), (64, 64, 8, 128, 1632, 3, 256), (17, 32, 8, 128, 4192, 5, 128)]


@pytest.mark.parametrize("T,nq,nkv,D,cap,splits,rows", NEIGHBOURS)
@pytest.mark.parametrize("at", [0, 2])
def test_other_lengths_move_nothing(lib, T, nq, nkv, D, cap, splits, rows, at):  # noqa: F811
    """One sequence of 1000 slots among three whose lengths change, out of range
    ones included."""
    c = Attn(lib, [1000] * 4, T, nq, nkv, D, "random", splits=splits, cap=cap, seed=T)
    assert group_rows(c, rows)
    seen = []
    for others in ([1000, 1000, 1000], [100, 100, 100], [0, -1, 1000], [1 << 30, 1000, 33], [-5, -5, -5], [1, 700, 31]):
        c.lens.copy_(i32(others[:at] + [1000] + others[at:]))
        c.out.fill_(3)
        c.run()
        torch.cuda.synchronize()
        seen.append(bits(c.rows()[at], c.kno[at], c.vno[at]))
    c.check([at])
    for s in seen[1:]:
        for x, y in zip(seen[0], s):
            assert torch.equal(x, y)


@pytest.mark.parametrize("T,nq,nkv,D,cap,splits,rows", [(3, 8, 2, 128, 4096, 1, 16), (4, 8, 8, 64, 4096, 2, 16),
                                                        (16, 32, 8, 128, 2080, 1, 32), (27, 32, 8, 128, 12256, 2, 128),
                                                        (64, 64, 8, 128, 3200, 1, 256)])
def test_other_rows_move_nothing(lib, T, nq, nkv, D, cap, splits, rows):  # noqa: F811
    """The last node's query changes: only its own rows do.  Scores of the cache
    grow with the slot, by more than the running maximum's slack again and again,
    at different slots for different rows."""
    L = 1500
    c = Attn(lib, [L] * 4, T, nq, nkv, D, "star", splits=splits, cap=cap, seed=D + T)
    assert group_rows(c, rows)
    c.k[:, :, :L] *= torch.linspace(0.1, 6, L, device=DEV)[None, None, :, None].to(torch.bfloat16)
    x = c.qkv.view(4, T, nq + 2 * nkv, D)
    g = torch.Generator(device=DEV).manual_seed(1)
    seen = []
    for _ in range(6):
        c.run()
        c.check()
        seen.append(bits(c.rows()[:, :T - 1]))
        x[:, T - 1, :nq] = torch.randn((4, nq, D), generator=g, device=DEV).sign().to(torch.bfloat16)
    for s in seen[1:]:
        assert torch.equal(seen[0][0], s[0])
