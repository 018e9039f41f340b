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


def python_guards():
    """(name, call, the guard's message): each call passes every other check that comes before a launch
    except, on these CPU tensors, the one of the device."""
    import torch

    from litemind_b200 import ops

    f32, bf16, i32 = torch.float32, torch.bfloat16, torch.int32
    x, i, w = torch.zeros(4, 64), torch.zeros(4, 2, dtype=i32), torch.zeros(4, 2)
    rows, gain = torch.zeros(8, 64), torch.ones(64)
    plan = ops.SortPlan(torch.zeros(9, dtype=i32), i)
    e4, e2 = ops.MxTensor.empty((4, 64), "e4m3", "cpu"), ops.MxTensor.empty((3, 5, 64), "e2m1", "cpu")
    offsets = torch.zeros(4, dtype=i32)
    data, scales = torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 16, dtype=torch.uint8)
    return [
        ("quantise type", lambda: ops.mx_quantize(x.double(), "e2m1"), "values must be float32"),
        ("quantise format", lambda: ops.mx_quantize(x, "fp4"), "unknown MX format"),
        ("quantise columns", lambda: ops.mx_quantize(x.t(), "e2m1"), "values must be a matrix with contiguous"),
        ("quantise rows that repeat", lambda: ops.mx_quantize(x[:1].expand(4, 64), "e2m1"), "non-overlapping rows"),
        ("quantise vector", lambda: ops.mx_quantize(x[0], "e2m1"), "values must be a matrix, or contiguous"),
        ("quantise stack", lambda: ops.mx_quantize(torch.zeros(2, 64, 4).transpose(1, 2), "e2m1"), "contiguous with more dimensions"),
        ("quantise out shape", lambda: ops.mx_quantize(x[:3], "e4m3", out=e4), "out has another shape or format"),
        ("quantise out format", lambda: ops.mx_quantize(x, "e2m1", out=e4), "out has another shape or format"),
        ("matrix format", lambda: ops.MxTensor(data, scales, 64, "e5m2"), "unknown MX format"),
        ("matrix type", lambda: ops.MxTensor(data.int(), scales, 64, "e4m3"), "must be contiguous uint8"),
        ("matrix strides", lambda: ops.MxTensor(data[:, ::2], scales, 64, "e2m1"), "must be contiguous uint8"),
        ("matrix columns", lambda: ops.MxTensor(data, scales, 129, "e4m3"), "do not have the layout"),
        ("matrix pitch", lambda: ops.MxTensor(data[:, :64].contiguous(), scales, 64, "e4m3"), "do not have the layout"),
        ("matrix scales", lambda: ops.MxTensor(data, scales[:3], 64, "e4m3"), "do not have the layout"),
        ("product columns", lambda: ops.mx_matmul(e4, ops.MxTensor.empty((3, 5, 63), "e2m1", "cpu"), offsets), "with the same k"),
        ("product weights", lambda: ops.mx_matmul(e4, e4, None), "w 4-bit"),
        ("product stack of x", lambda: ops.mx_matmul(e2, e2, offsets), "x must be"),
        ("sort columns", lambda: ops.sort_rows(x.t(), plan), "x must be a matrix with contiguous"),
        ("sort tokens", lambda: ops.sort_rows(x[:3], plan), "a row for each token"),
        ("sort format", lambda: ops.sort_rows(e4, plan, out=ops.MxTensor.empty((8, 64), "e2m1", "cpu")), "format and columns"),
        ("plan type", lambda: ops.sort_plan(i.long(), 8), "topk_idx must be contiguous int32"),
        ("plan strides", lambda: ops.sort_plan(torch.zeros(2, 4, dtype=i32).t(), 8), "topk_idx must be contiguous int32"),
        ("plan experts", lambda: ops.sort_plan(i, 0), "experts must be in"),
        ("plan many experts", lambda: ops.sort_plan(i, 1025), "experts must be in"),
        ("plan of other types", lambda: ops.SortPlan(torch.zeros(9), i), "offsets must be int32"),
        ("plan of matrices", lambda: ops.SortPlan(i, i), "offsets must be int32"),
        ("back rows", lambda: ops.unsort_rows(rows.t(), plan), "rows must be a contiguous matrix"),
        ("back type", lambda: ops.unsort_rows(rows.double(), plan), "rows must be float32"),
        ("back weights", lambda: ops.unsort_rows(rows, plan, torch.zeros(4, 3)), "weights must be contiguous float32"),
        ("back weights type", lambda: ops.unsort_rows(rows, plan, w.half()), "weights must be contiguous float32"),
        ("back to nothing", lambda: ops.unsort_rows(rows, plan, accumulate=True), "accumulate needs out"),
        ("back to another type", lambda: ops.unsort_rows(rows, plan, dtype=torch.float16), "rows' type or float32"),
        ("back to an out of another type", lambda: ops.unsort_rows(rows, plan, out=x.to(bf16)), "rows' type or float32"),
        ("back to another shape", lambda: ops.unsort_rows(rows, plan, out=x[:3]), "out must be contiguous"),
        ("gradient rows", lambda: ops.unsort_rows_backward(x, rows.t(), plan, w), "rows must be a contiguous matrix"),
        ("gradient tokens", lambda: ops.unsort_rows_backward(x[:3], rows, plan, w), "grad_y must be contiguous"),
        ("gradient type", lambda: ops.unsort_rows_backward(x.half(), rows, plan, w), "rows' type or float32"),
        ("gradient other type", lambda: ops.unsort_rows_backward(x.half(), rows.to(bf16), plan, w), "rows' type or float32"),
        ("gradient weights", lambda: ops.unsort_rows_backward(x, rows, plan, w[:, :1]), "weights must be contiguous float32"),
        ("norm type", lambda: ops.add_rms_norm(x.half(), None, gain, 1e-6), "hidden must be contiguous"),
        ("norm vector", lambda: ops.add_rms_norm(x[0], None, gain, 1e-6), "hidden must be contiguous"),
        ("norm delta shape", lambda: ops.add_rms_norm(x, x[:2], gain, 1e-6), "delta must be contiguous"),
        ("norm delta type", lambda: ops.add_rms_norm(x, x.half(), gain, 1e-6), "delta must be contiguous"),
        ("norm weight", lambda: ops.add_rms_norm(x, None, gain[:63], 1e-6), "weight must be contiguous"),
        ("norm weight type", lambda: ops.add_rms_norm(x, None, gain.to(bf16), 1e-6), "weight must be contiguous"),
        ("norm format", lambda: ops.add_rms_norm(x, None, gain, 1e-6, fmt="e5m2"), "unknown MX format"),
        # the device, one for each call
        ("quantise on the CPU", lambda: ops.mx_quantize(x, "e2m1"), "on a CUDA device"),
        ("dequantise on the CPU", lambda: ops.mx_dequantize(e4), "on a CUDA device"),
        ("product on the CPU", lambda: ops.mx_matmul(e4, e2, offsets), "on a CUDA device"),
        ("plan on the CPU", lambda: ops.sort_plan(i, 8), "on a CUDA device"),
        ("sort on the CPU", lambda: ops.sort_rows(x, plan), "on a CUDA device"),
        ("back on the CPU", lambda: ops.unsort_rows(rows, plan, w), "on a CUDA device"),
        ("gradient on the CPU", lambda: ops.unsort_rows_backward(x, rows, plan, w), "on a CUDA device"),
        ("norm on the CPU", lambda: ops.add_rms_norm(x, x, gain, 1e-6), "on a CUDA device"),
    ]


@pytest.mark.parametrize("case", range(54))
def test_python_guards(case):
    """Each guard by its own message: with the guard taken out another check would answer."""
    pytest.importorskip("torch")
    cases = python_guards()
    assert len(cases) == 54
    name, call, message = cases[case]
    with pytest.raises(ValueError, match=message):
        call()
        pytest.fail(f"{name} was not refused")


def test_gradient_entry_by_types(monkeypatch):
    """Only 16-bit rows with a float32 grad_y take the entry for it; messages name the entry that was called."""
    torch = pytest.importorskip("torch")
    from litemind_b200 import ops

    called = []
    monkeypatch.setattr(ops, "_index", lambda *tensors: 0)
    monkeypatch.setattr(ops, "_call", lambda fn, *args: called.append(fn.__name__))
    plan = ops.SortPlan(torch.zeros(9, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32))
    for rows_type, grad_type in ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float32)):
        ops.unsort_rows_backward(torch.zeros(4, 8, dtype=grad_type), torch.zeros(8, 8, dtype=rows_type), plan, torch.zeros(4, 2))
    name = "lm_moe_unsort_rows_backward"
    assert called == [name, name, name + "_f32", name + "_f32"]
