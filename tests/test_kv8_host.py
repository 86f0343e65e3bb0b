"""What the engine refuses beside an 8-bit cache, before it touches a device."""

import pytest

import engine


@pytest.mark.parametrize("kw", [dict(kv_cache="fp8"), dict(kv_cache=None), dict(kv_cache=True), dict(kv_cache=["int8"]),
                                dict(kv_cache="int8", speculate="tree"), dict(kv_cache="int8", mega=True),
                                dict(kv_cache="int8", speculate="chain")], ids=str)
def test_engine_refuses(kw):
    with pytest.raises(ValueError, match="kv_cache|speculate"):
        engine.Engine("/nowhere", **kw)
    with pytest.raises(ValueError, match="kv_cache|speculate"):
        engine.Engine.from_tensors({}, {}, **kw)


def test_modes_that_go_together():
    for kv in ("bf16", "int8"):
        engine.check_modes(kv, False, None)
        engine.check_modes(kv, True, False)
    engine.check_modes("bf16", "tree", None)
    engine.check_modes("bf16", False, True)


def test_splits_of_a_state():
    from qdec.runtime import kv8_splits
    for shape, n in (((1, 8, 512), 0), ((1, 8, 640), 3), ((1, 8, 1024), 4), ((1, 8, 1152), 0), ((8, 8, 1024), 4), ((9, 8, 1024), 0),
                     ((32, 2, 640), 3), ((32, 8, 640), 0)):
        assert kv8_splits(*shape) == n, shape
