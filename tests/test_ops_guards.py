"""What the stand-alone operators refuse, each case held to its own message, without a GPU: through
the C ABI with addresses that overlap nowhere unless the case says so, and through litemind_b200.ops
with the guard that each case is for."""
import pytest

from litemind_b200 import _lib

BAD, OK = _lib.LM_ERR_INVALID_ARGUMENT, _lib.LM_OK


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_debug_knobs(lib):
    for knob, value in ((1, 0), (99, 0), (_lib.LM_DEBUG_WAIT_LIMIT_NS, -1), (_lib.LM_DEBUG_WAIT_LIMIT_NS, 2 * 10**9 + 1),
                        (_lib.LM_DEBUG_PRODUCT_STALL, -1), (_lib.LM_DEBUG_PRODUCT_STALL, _lib.LM_STALL_TMEM_EMPTY + 1)):
        assert lib.lm_ops_debug_set(knob, value) == BAD
        assert lib.lm_moe_last_error(None).decode().startswith("lm_ops_debug_set:")
    for knob, value in ((_lib.LM_DEBUG_WAIT_LIMIT_NS, 1000), (_lib.LM_DEBUG_WAIT_LIMIT_NS, 0), (_lib.LM_DEBUG_PRODUCT_STALL, 3), (_lib.LM_DEBUG_PRODUCT_STALL, 0)):
        assert lib.lm_ops_debug_set(knob, value) == OK


def test_sync_asks_the_device_it_names(monkeypatch):
    """A device without an index is the current one, not device 0."""
    torch = pytest.importorskip("torch")
    from litemind_b200 import ops

    asked = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(ops, "_call", lambda fn, index, *args: asked.append(index))
    for device in (None, "cuda", torch.device("cuda"), "cuda:0", "cuda:1", torch.device("cuda", 2)):
        ops.sync(device)
    assert asked == [3, 3, 3, 0, 1, 2]
    with pytest.raises(ValueError, match="CUDA device"):
        ops.sync("cpu")


def refused(lib, name, message, good, *changes):
    """Each change turns the call into one that is refused with this message (`good` itself is never
    made: its addresses hold nothing)."""
    order = list(good)
    for change in changes:
        args = dict(good, **change)
        assert getattr(lib, name)(*[args[o] for o in order], None) == BAD, (name, change)
        assert message in lib.lm_moe_last_error(None).decode(), (name, change, lib.lm_moe_last_error(None))


def places(*names):
    """An address for each, 2^32 apart."""
    return {name: (i + 1) << 32 for i, name in enumerate(names)}


def test_sort_overlaps(lib):
    good = dict(places("idx"), tokens=100, k=6, experts=64, **places("_", "offsets", "at"))
    del good["_"]
    idx, offsets, at = good["idx"], good["offsets"], good["at"]
    refused(lib, "lm_moe_sort_plan", "overlap", good, dict(at=idx), dict(at=idx + 2396), dict(at=idx - 2396), dict(offsets=idx), dict(offsets=idx - 256),
            dict(offsets=idx + 2396), dict(offsets=at + 4), dict(offsets=at - 256))
    a = places("x", "at", "rows")
    good = dict(x=a["x"], xstride=256, at=a["at"], tokens=5, k=2, bytes=128, rows=a["rows"], rstride=256, n=10)
    x, at = a["x"], a["at"]
    refused(lib, "lm_moe_sort_rows", "overlaps", good, dict(rows=x), dict(rows=x + 127), dict(rows=x - 127), dict(rows=x + 4 * 256 + 127), dict(rows=x - 9 * 256),
            dict(rows=x + 2, rstride=2**40), dict(rows=x, rstride=128), dict(rows=x - 64, rstride=128, n=1), dict(rows=x + 1000, rstride=512), dict(rows=at), dict(rows=at + 39),
            dict(rows=at - 9 * 256 - 127), dict(rows=x, xstride=2**60, rstride=2**61))
