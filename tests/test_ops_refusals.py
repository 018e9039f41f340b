"""What the stand-alone operators refuse, through the C ABI without a GPU: every bad argument is
answered with a status and a message before anything is launched, and empty inputs are no error."""
import subprocess

import pytest

from litemind_b200 import _lib

BAD, OK = _lib.LM_ERR_INVALID_ARGUMENT, _lib.LM_OK
P = 1 << 20  # an aligned address that is never read
F32, BF16, F16 = _lib.LM_DTYPE_F32, _lib.LM_DTYPE_BF16, _lib.LM_DTYPE_F16
E2M1, E4M3 = _lib.LM_MX_E2M1, _lib.LM_MX_E4M3


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, name, good, **changes):
    """Each change alone turns the good call into a refused one with a message that names the entry."""
    order = list(good)
    for key, values in changes.items():
        for v in values:
            args = dict(good, **{key: v})
            assert getattr(lib, name)(*[args[o] for o in order], None) == BAD, (name, key, v)
            assert lib.lm_moe_last_error(None).decode().startswith(name + ":"), (key, v)


def empty(lib, name, good, **changes):
    order = list(good)
    for key, values in changes.items():
        for v in values:
            args = dict(good, **{key: v})
            assert getattr(lib, name)(*[args[o] for o in order], None) == OK, (name, key, v)


def test_pitches(lib):
    assert [lib.lm_mx_data_pitch(E2M1, c) for c in (0, 1, 128, 129, 1408)] == [0, 64, 64, 128, 704]
    assert [lib.lm_mx_data_pitch(E4M3, c) for c in (0, 1, 128, 129, 1408)] == [0, 128, 128, 256, 1408]
    assert [lib.lm_mx_scale_pitch(c) for c in (0, 1, 512, 513, 2048)] == [0, 16, 16, 32, 64]
    assert lib.lm_mx_data_pitch(9, 10) == 0 and lib.lm_mx_data_pitch(E2M1, -1) == 0 and lib.lm_mx_scale_pitch(-1) == 0
    assert lib.lm_mx_scale_pitch(2**24 + 1) == 0


def test_quantise(lib):
    good = dict(values=P, dtype=BF16, rows=4, cols=100, stride=100, fmt=E2M1, data=P, scales=P)
    refused(lib, "lm_mx_quantize", good, values=[None, P + 1], dtype=[0, 4, -1], rows=[-1, 2**31], cols=[-1, 2**24 + 1], stride=[99, -1], fmt=[0, 3],
            data=[None, P + 16], scales=[None, P + 8])
    empty(lib, "lm_mx_quantize", good, rows=[0], cols=[0])


def test_dequantise(lib):
    good = dict(data=P, scales=P, fmt=E4M3, rows=4, cols=100, values=P, dtype=F32, stride=100)
    refused(lib, "lm_mx_dequantize", good, values=[None, P + 2], dtype=[0, 4], rows=[-1], cols=[-1, 2**24 + 1], stride=[99], fmt=[0, 3],
            data=[None, P + 16], scales=[None, P + 8])
    empty(lib, "lm_mx_dequantize", good, rows=[0], cols=[0])


def test_product(lib):
    good = dict(x=P, xs=P, fmt=E4M3, rows=10, w=P, ws=P, groups=4, n=64, k=100, offsets=P, out=P, dtype=BF16, stride=64)
    refused(lib, "lm_mx_matmul", good, x=[None, P + 16], xs=[None, P + 8], fmt=[0, 3], rows=[-1, 2**31], w=[None, P + 16], ws=[None, P + 4], groups=[0, -1, 1025],
            n=[-1, 2**30], k=[-1, 0, 2**24 + 1], offsets=[None, P + 2], out=[None, P + 1], dtype=[0, 4], stride=[63])
    empty(lib, "lm_mx_matmul", good, rows=[0], n=[0])


def test_norm(lib):
    good = dict(hidden=P, dtype=F32, delta=P, ddtype=BF16, weight=P, rows=3, count=100, eps=1e-6, sum=P, bf16=P, fmt=E4M3, data=P, scales=P)
    refused(lib, "lm_gemm_add_rms_norm_mx", good, hidden=[None, P + 2], dtype=[0, F16], delta=[P + 1], ddtype=[F16], weight=[None, P + 2], rows=[-1, 2**31],
            count=[-1, 2**24 + 1], eps=[-1.0, float("nan")], sum=[None, P + 2], bf16=[P + 1], fmt=[0, 3], data=[None, P + 16], scales=[None, P + 8])
    empty(lib, "lm_gemm_add_rms_norm_mx", good, rows=[0], count=[0])


def test_sort(lib):
    good = dict(idx=P, tokens=5, k=6, experts=64, offsets=P, at=P)
    refused(lib, "lm_moe_sort_plan", good, idx=[None, P + 1], tokens=[-1, 2**30], k=[0, 65], experts=[0, 1025], offsets=[None, P + 2], at=[None, P + 2])
    good = dict(x=P, xstride=128, at=P, tokens=5, k=6, bytes=128, rows=P, rstride=128, n=30)
    refused(lib, "lm_moe_sort_rows", good, x=[None], xstride=[127], at=[None, P + 1], tokens=[-1, 2**30], k=[0, 65], bytes=[-1], rows=[None], rstride=[127], n=[-1])
    empty(lib, "lm_moe_sort_rows", good, tokens=[0], bytes=[0], n=[0])
    good = dict(rows=P, dtype=BF16, n=30, at=P, weights=P, tokens=5, k=6, cols=64, y=P, ydtype=F32, acc=0)
    refused(lib, "lm_moe_unsort_rows", good, rows=[None, P + 1], dtype=[0, 4], n=[-1], at=[None, P + 2], weights=[P + 1], tokens=[-1, 2**30], k=[0, 65],
            cols=[-1, 2**24 + 1], y=[None, P + 2], ydtype=[F16, 0])
    empty(lib, "lm_moe_unsort_rows", good, tokens=[0], cols=[0])
    good = dict(gy=P, rows=P, dtype=F16, n=30, at=P, weights=P, tokens=5, k=6, cols=64, gr=P, gw=P)
    refused(lib, "lm_moe_unsort_rows_backward", good, gy=[None, P + 1], rows=[None, P + 1], dtype=[0, 4], n=[-1], at=[None, P + 2], weights=[None, P + 1],
            tokens=[-1, 2**30], k=[0, 65], cols=[-1, 2**24 + 1], gr=[None, P + 1], gw=[None, P + 2])
    empty(lib, "lm_moe_unsort_rows_backward", good, tokens=[0])


def test_overlaps(lib):
    at, far = 1 << 30, 1 << 32
    back = dict(rows=P, dtype=BF16, n_rows=6, at=at, weights=at, tokens=3, k=2, cols=64, y=far, y_dtype=BF16, accumulate=0)
    refused(lib, "lm_moe_unsort_rows", back, y=[P, P + 6 * 128 - 2, P - 3 * 128 + 2])
    grad = dict(grad_y=P, rows=far, dtype=BF16, n_rows=6, at=at, weights=at, tokens=3, k=2, cols=64, grad_rows=far, grad_weights=at)
    refused(lib, "lm_moe_unsort_rows_backward", grad, grad_rows=[P, P + 3 * 128 - 16, far + 128, far - 6 * 128 + 16])
    norm = dict(hidden=P, dtype=F32, delta=far, ddtype=BF16, weight=at, rows=4, count=64, eps=1e-6, sum=2 * far, bf16=None, fmt=E4M3, data=at, scales=at)
    refused(lib, "lm_gemm_add_rms_norm_mx", norm, sum=[P + 256, P - 256, far, far + 4 * 128 - 16])


def test_cpp_forms(tmp_path):
    """Mx.hpp and TokenSort.hpp compile as a user compiles them and answer as the C entries do."""
    from tests.test_cpp_mirror import _compile

    res = subprocess.run([_compile("MxTest", tmp_path)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout + res.stderr


def test_python_checks():
    """litemind_b200.ops refuses with ValueError, on CPU tensors too."""
    torch = pytest.importorskip("torch")
    from litemind_b200 import ops

    x, i = torch.zeros(4, 64), torch.zeros(4, 2, dtype=torch.int32)
    u8 = torch.zeros(4, 64, dtype=torch.uint8)
    s16 = torch.zeros(4, 16, dtype=torch.uint8)
    cases = [lambda: ops.mx_quantize(x, "e2m1"), lambda: ops.mx_quantize(x, "fp4"), lambda: ops.mx_quantize(x.double(), "e2m1"), lambda: ops.mx_quantize(x.t(), "e2m1"),
             lambda: ops.mx_quantize(x[0], "e2m1"), lambda: ops.MxTensor(u8, s16, 129, "e2m1"), lambda: ops.MxTensor(u8, s16, 64, "e4m3"),
             lambda: ops.MxTensor(u8.int(), s16, 64, "e2m1"), lambda: ops.MxTensor(u8, s16[:, :8], 64, "e2m1"), lambda: ops.sort_plan(i, 8), lambda: ops.sort_plan(i.long(), 8),
             lambda: ops.sort_plan(i, 0), lambda: ops.SortPlan(i, i), lambda: ops.mx_dequantize(ops.MxTensor(u8, s16, 64, "e2m1")),
             lambda: ops.mx_matmul(ops.MxTensor(u8, s16, 64, "e2m1"), ops.MxTensor(u8, s16, 63, "e2m1")),
             lambda: ops.mx_matmul(ops.MxTensor(u8, s16, 64, "e2m1"), ops.MxTensor(u8, s16, 64, "e2m1")),
             lambda: ops.add_rms_norm(x, x, torch.zeros(64), 1e-6), lambda: ops.add_rms_norm(x, x[:2], torch.zeros(64), 1e-6),
             lambda: ops.add_rms_norm(x.half(), None, torch.zeros(64), 1e-6), lambda: ops.add_rms_norm(x, None, torch.zeros(63), 1e-6)]
    plan = ops.SortPlan(torch.zeros(9, dtype=torch.int32), i)
    cases += [lambda: ops.sort_rows(x[:3], plan), lambda: ops.sort_rows(x, plan), lambda: ops.unsort_rows(x, plan, torch.zeros(4, 3)),
              lambda: ops.unsort_rows(x, plan, accumulate=True), lambda: ops.unsort_rows(x, plan, dtype=torch.float16),
              lambda: ops.unsort_rows_backward(x[:3], x, plan, torch.zeros(4, 2)), lambda: ops.unsort_rows_backward(x.half(), x, plan, torch.zeros(4, 2)),
              lambda: ops.unsort_rows_backward(x, x, plan, torch.zeros(4, 2))]
    for n, case in enumerate(cases):
        with pytest.raises(ValueError):
            case()
            pytest.fail(f"case {n} was not refused")
