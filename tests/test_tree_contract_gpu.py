"""What a result of the tree attention depends on: the splits, its sequence's
length and the call's shape.  The other sequences' lengths do not move its bits."""

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
