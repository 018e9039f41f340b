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


def test_mx_overlaps(lib):
    a = places("values", "data", "scales")
    v, d, s = a["values"], a["data"], a["scales"]
    good = dict(values=v, dtype=_lib.LM_DTYPE_BF16, rows=4, cols=100, stride=200, fmt=_lib.LM_MX_E4M3, data=d, scales=s)
    refused(lib, "lm_mx_quantize", "overlap", good, dict(data=v), dict(data=v + 1376), dict(data=v - 3 * 128), dict(data=v - 480), dict(scales=v), dict(scales=v + 3 * 400 + 192),
            dict(scales=v - 48), dict(scales=d), dict(scales=d + 496), dict(data=s + 32), dict(data=s - 480))
    good = dict(data=d, scales=s, fmt=_lib.LM_MX_E2M1, rows=4, cols=100, values=v, dtype=_lib.LM_DTYPE_F32, stride=100)
    refused(lib, "lm_mx_dequantize", "overlaps", good, dict(values=d), dict(values=d + 252), dict(values=d - 1596), dict(values=s), dict(values=s + 60), dict(values=s - 1596))
    a = places("x", "xs", "w", "ws", "offsets", "out")
    good = dict(x=a["x"], xs=a["xs"], fmt=_lib.LM_MX_E4M3, rows=10, w=a["w"], ws=a["ws"], groups=4, n=64, k=100, offsets=a["offsets"], out=a["out"], dtype=_lib.LM_DTYPE_F32, stride=80)
    size = dict(x=1280, xs=160, w=256 * 64, ws=256 * 16, offsets=20)
    refused(lib, "lm_mx_matmul", "out overlaps an input", good, *[dict(out=a[i] + by) for i in size for by in (0, size[i] - 4, -9 * 320 - 252)])


def test_norm_overlaps(lib):
    a = places("hidden", "delta", "weight", "sum", "bf16", "data", "scales")
    size = dict(hidden=4 * 64 * 4, delta=4 * 64 * 2, weight=256, sum=4 * 64 * 4, bf16=4 * 64 * 2, data=4 * 128, scales=4 * 16)
    good = dict(hidden=a["hidden"], dtype=_lib.LM_DTYPE_F32, delta=a["delta"], ddtype=_lib.LM_DTYPE_BF16, weight=a["weight"], rows=4, count=64, eps=1e-6, sum=a["sum"],
                bf16=a["bf16"], fmt=_lib.LM_MX_E4M3, data=a["data"], scales=a["scales"])
    for out in ("bf16", "data", "scales"):
        refused(lib, "lm_gemm_add_rms_norm_mx", "overlap", good, *[{out: a[i] + by} for i in a if i != out for by in (0, (size[i] - 1) // 32 * 32, -((size[out] - 1) // 32 * 32))])
    refused(lib, "lm_gemm_add_rms_norm_mx", "overlap", good, *[dict(sum=a["weight"] + by) for by in (0, 252, -1020)])


def test_way_back_overlaps(lib):
    a = places("rows", "at", "weights", "y")
    good = dict(rows=a["rows"], dtype=_lib.LM_DTYPE_BF16, n=6, at=a["at"], weights=a["weights"], tokens=3, k=2, cols=64, y=a["y"], ydtype=_lib.LM_DTYPE_F32, acc=0)
    size = dict(rows=6 * 128, at=24, weights=24)
    refused(lib, "lm_moe_unsort_rows", "y overlaps", good, *[dict(y=a[i] + by) for i in size for by in (0, size[i] - 4, 4 - 3 * 256)])
    a = places("gy", "rows", "at", "weights", "gr", "gw")
    good = dict(gy=a["gy"], rows=a["rows"], dtype=_lib.LM_DTYPE_F16, n=6, at=a["at"], weights=a["weights"], tokens=3, k=2, cols=64, gr=a["gr"], gw=a["gw"])
    size = dict(gy=3 * 128, rows=6 * 128, at=24, weights=24, gr=6 * 128)
    refused(lib, "lm_moe_unsort_rows_backward", "overlap", good, *[dict(gw=a[i] + by) for i in size for by in (0, size[i] - 4, -20)],
            *[dict(gr=a[i] + by) for i in ("gy", "at", "weights", "gw") for by in (0, 20, 4 - 6 * 128)], dict(gr=a["rows"] + 128), dict(gr=a["rows"] - 128))


def test_gradient_of_an_f32_result(lib):
    """lm_moe_unsort_rows_backward_f32 refuses what its sibling refuses, with f32's alignment and size."""
    a = places("gy", "rows", "at", "weights", "gr", "gw")
    good = dict(gy=a["gy"], rows=a["rows"], dtype=_lib.LM_DTYPE_BF16, n=6, at=a["at"], weights=a["weights"], tokens=3, k=2, cols=64, gr=a["gr"], gw=a["gw"])
    name = "lm_moe_unsort_rows_backward_f32"
    refused(lib, name, name + ": tensors are", good, dict(dtype=0), dict(dtype=4))
    refused(lib, name, name + ": a size", good, dict(n=-1), dict(tokens=-1), dict(tokens=2**30), dict(k=0), dict(k=65), dict(cols=-1), dict(cols=2**24 + 1))
    refused(lib, name, name + ": a null or misaligned", good, dict(gy=None), dict(gy=a["gy"] + 2), dict(rows=None), dict(rows=a["rows"] + 1), dict(at=None), dict(at=a["at"] + 2),
            dict(weights=None), dict(weights=a["weights"] + 2), dict(gr=None), dict(gr=a["gr"] + 1), dict(gw=None), dict(gw=a["gw"] + 2))
    refused(lib, name, name + ": grad_rows overlaps", good, dict(gr=a["gy"]), dict(gr=a["gy"] + 3 * 256 - 2), dict(gr=a["rows"] + 128))
    refused(lib, name, name + ": grad_rows and grad_weights", good, dict(gw=a["gy"] + 3 * 256 - 4), dict(gw=a["rows"]), dict(gw=a["weights"]), dict(gr=a["at"]))
    order = list(good)
    assert getattr(lib, name)(*[dict(good, tokens=0)[o] for o in order], None) == OK


def test_cpp_forms_take_every_type_and_stride(tmp_path):
    import subprocess

    from tests.test_cpp_mirror import _compile

    res = subprocess.run([_compile("OpsFormsTest", tmp_path)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout + res.stderr
