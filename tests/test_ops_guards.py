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
