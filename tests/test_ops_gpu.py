"""The operators of litemind_b200.ops on the GPU against 64-bit implementations of their formulas
(tests/mx_reference.py): MX matrices and their grouped product, the residual norm with an MX
output, tokens sorted by expert and back with both gradients, and a feed-forward made of them.

Tolerances are derived, not fitted.  Quantisation and the sort are exact.  A sum of n terms in f32
is off by at most n 2^-23 of the sum of the terms' magnitudes (2^-23: an adder that truncates), and
a result rounded to a type by half a step, finfo.eps / 2 of it.
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from litemind_b200 import ops  # noqa: E402
from tests import mx_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Below the least normal number steps no longer shrink."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def same_bits(a, b):
    assert a.shape == b.shape and a.dtype == b.dtype
    kind = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    assert torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


# ---------------------------------------------------------------- MX matrices

SIZES = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 127), (4, 128), (7, 129), (3, 511), (2, 513), (65, 1413), (1, 2048), (33, 4100)]


def check_quantised(q, x, fmt):
    codes, byte, values = ref.quantise(x.double(), fmt)
    data, scales = ref.layout(codes, byte, fmt)
    assert torch.equal(q.scales, scales)
    assert torch.equal(q.data, data)
    return values


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantise_and_back(rows, cols, dtype, fmt):
    g = gen(rows * 7919 + cols)
    x = (normal(g, rows, cols) * torch.exp2(4 * normal(g, rows, 1))).to(dtype)
    x[:, ::5] = 0
    q = ops.mx_quantize(x, fmt)
    values = check_quantised(q, x, fmt)
    for out in (F32, BF16, F16):
        got = ops.mx_dequantize(q, out)
        assert got.dtype == out
        assert torch.equal(got, values.to(out))


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_quantise_ties_ends_and_signs(fmt):
    """Every midpoint of the format's values (ties go to even), values past the last one, the
    extremes of f32, negative zero, and blocks of zeros."""
    grid = ref.E2M1 if fmt == "e2m1" else ref.E4M3
    mid = (grid[1:] + grid[:-1]) / 2
    top = float(grid[-1])
    points = torch.cat((grid, mid, torch.tensor([top * 1.05, top * 1.1]))).float()
    rows = []
    for v in points.tolist():
        block = [v, -v] + [0.0, -0.0] * 14 + [top, -top]  # the last two fix the scale at 1
        for s in (1.0, 2.0**-100, 2.0**100):
            rows.append([b * s for b in block])
    big = torch.finfo(F32).max
    rows += [[big, -big, 1.0] + [0.0] * 29, [2.0**-149, -(2.0**-149)] + [0.0] * 30, [2.0**-126, 2.0**-127] + [2.0**-130] * 30,
             [0.0] * 32, [-0.0] * 32, [2.0**-120] * 32, [2.0**-125, 2.0**-119] * 16]
    x = torch.tensor(rows, dtype=F32, device="cuda")
    q = ops.mx_quantize(x, fmt)
    values = check_quantised(q, x, fmt)
    assert torch.equal(ops.mx_dequantize(q, F32), values.float())


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_quantise_nan_block(bad, fmt):
    """A NaN or an infinity makes its own block NaN and no other."""
    x = normal(gen(3), 3, 100)
    x[1, 40] = bad
    q = ops.mx_quantize(x, fmt)
    check_quantised(q, x, fmt)
    back = ops.mx_dequantize(q, F32)
    assert torch.isnan(back[1, 32:64]).all()
    back[1, 32:64] = 0
    assert torch.isfinite(back).all()


def test_quantise_strides_and_stacks():
    g = gen(5)
    wide = normal(g, 6, 300, dtype=BF16)
    for view in (wide[:, 3:200], wide[::2], wide[1:2], wide[:, :40], wide.view(-1)[1:1601].view(8, 200)):
        check_quantised(ops.mx_quantize(view, "e2m1"), view, "e2m1")
    stack = normal(g, 2, 3, 100)
    q = ops.mx_quantize(stack, "e4m3")
    assert q.shape == (2, 3, 100)
    flat = ops.mx_quantize(stack.view(6, 100), "e4m3")
    assert torch.equal(q.data.view(6, -1), flat.data) and torch.equal(q.scales.view(6, -1), flat.scales)
    assert torch.equal(ops.mx_dequantize(q), ops.mx_dequantize(flat).view(2, 3, 100))


def test_quantise_past_32_bits():
    """Offsets past 2^31 elements: the last rows of a large matrix."""
    rows, cols = 1100000, 2048
    x = torch.zeros(rows, cols, dtype=F16, device="cuda")
    x[-5:] = normal(gen(8), 5, cols, dtype=F16)
    q = ops.mx_quantize(x, "e4m3")
    tail = ops.MxTensor(q.data[-5:].contiguous(), q.scales[-5:].contiguous(), cols, "e4m3")
    check_quantised(tail, x[-5:], "e4m3")
    assert torch.equal(ops.mx_dequantize(q, F16)[-5:], ops.mx_dequantize(tail, F16))


# ---------------------------------------------------------------- the grouped product


def product_inputs(seed, counts, n, k, fmt, extra=0):
    g = gen(seed)
    groups, rows = len(counts), sum(counts) + extra
    x = ops.mx_quantize(normal(g, rows, k) * torch.exp2(normal(g, rows, 1)), fmt)
    w = ops.mx_quantize(normal(g, groups, n, k) * 0.05, "e2m1")
    cut = [0]
    for c in counts:
        cut.append(cut[-1] + c)
    return x, w, torch.tensor(cut, dtype=torch.int32, device="cuda"), cut


def check_product(out, x, w, cut, k, dtype):
    xv, wv = ref.values(x.data, x.scales, k, x.fmt), ref.values(w.data, w.scales, k, "e2m1")
    for g, (a, b) in enumerate(zip(cut, cut[1:])):
        if b > a:
            want, size = xv[a:b] @ wv[g].t(), xv[a:b].abs() @ wv[g].abs().t()
            off = (out[a:b].double() - want).abs()
            assert (off <= k * 2.0**-23 * size + half_step(dtype) * want.abs() * 1.001 + tiny(dtype)).all(), (g, a, b, off.max())


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,n,k", [
    ([1], 1, 1), ([1], 128, 128), ([3], 130, 33), ([17], 64, 100), ([128], 256, 512), ([129], 127, 640), ([300], 384, 1408),
    ([1, 0, 2, 0], 72, 96), ([0, 0, 0, 5], 200, 260), ([16, 17, 15, 1, 0, 33], 257, 1413), ([200, 1, 0, 130], 128, 2048),
    ([1] * 64, 96, 64), ([2, 5, 9] * 20, 320, 160), ([64, 0, 0, 640, 1], 500, 1152)])
def test_product(counts, n, k, dtype, fmt):
    x, w, offsets, cut = product_inputs(n + k, counts, n, k, fmt)
    check_product(ops.mx_matmul(x, w, offsets, dtype=dtype), x, w, cut, k, dtype)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 96, 127, 128, 200, 255, 256, 257, 1000])
@pytest.mark.parametrize("k", [96, 2048])
def test_product_one_group(rows, k):
    """Every choice of the kernel's tile, with and without a ragged edge; no offsets needed."""
    x, w, _, cut = product_inputs(rows, [rows], 300, k, "e4m3")
    out = ops.mx_matmul(x, ops.MxTensor(w.data[0], w.scales[0], k, "e2m1"), dtype=BF16)
    check_product(out, x, w, cut, k, BF16)


def test_product_expert_layer_shapes():
    """The gate/up and down products of a 64-expert layer with ragged loads, empty experts among them."""
    counts = [(e * 37) % 61 if e % 5 else 0 for e in range(64)]
    for n, k in ((2816, 2048), (2048, 1408)):
        x, w, offsets, cut = product_inputs(n, counts, n, k, "e4m3")
        check_product(ops.mx_matmul(x, w, offsets, dtype=F32), x, w, cut, k, F32)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,n,k", [([4096], 4864, 300), ([700, 130, 0, 1, 1221, 128, 129, 1787], 4740, 1413), ([200] * 32, 3000, 1024), ([1000, 3100], 5001, 96)])
def test_product_many_rows(counts, n, k, dtype, fmt):
    """Enough rows a group and tiles for pairs of CTAs: ragged ends on every axis."""
    x, w, offsets, cut = product_inputs(n + k, counts, n, k, fmt)
    check_product(ops.mx_matmul(x, w, offsets, dtype=dtype), x, w, cut, k, dtype)


@pytest.mark.parametrize("rows", [1, 5, 16, 17, 40, 64, 100, 128])
@pytest.mark.parametrize("k", [1000, 1024, 2100, 4000, 10944])
def test_product_long_columns(rows, k):
    """Few tiles of many columns: clusters share a tile and add their sums, equal from call to call."""
    for counts, n in (([rows], 200), ([rows, 0, 3], 130)):
        x, w, offsets, cut = product_inputs(rows + k, counts, n, k, "e4m3")
        out = ops.mx_matmul(x, w, offsets, dtype=F32)
        check_product(out, x, w, cut, k, F32)
        same_bits(ops.mx_matmul(x, w, offsets, dtype=F32), out)
        for dtype in (BF16, F16):
            check_product(ops.mx_matmul(x, w, offsets, dtype=dtype), x, w, cut, k, dtype)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("counts", [[1], [7], [17], [31], [33], [60], [65], [100], [129], [1, 0, 6], [50, 49], [3, 60, 1]])
def test_product_few_rows_after_nan(counts, fmt):
    """Fewer rows than a tile has room for, in every CTA: what an earlier product left in shared memory
    and TMEM, NaN here, reaches nothing.  Also packed rows of many columns, shared by a cluster."""
    n, k = 148 * 128 // len(counts), 640
    x, w, offsets, cut = product_inputs(sum(counts), counts, n, k, fmt)
    nan = ops.MxTensor(torch.full((300, x.data.shape[1]), 0x7F, dtype=torch.uint8, device="cuda"), torch.full((300, x.scales.shape[1]), 255, dtype=torch.uint8, device="cuda"),
                       k, fmt)
    flat = ops.MxTensor(w.data.view(-1, w.data.shape[-1]), w.scales.view(-1, w.scales.shape[-1]), k, "e2m1")
    for rows in (16, 32, 64, 300):
        assert torch.isnan(ops.mx_matmul(ops.MxTensor(nan.data[:rows], nan.scales[:rows], k, fmt), flat, dtype=F32)).all()
        check_product(ops.mx_matmul(x, w, offsets, dtype=F32), x, w, cut, k, F32)
    x, w, offsets, cut = product_inputs(7, counts, 130, 6000, fmt)
    check_product(ops.mx_matmul(x, w, offsets, dtype=BF16), x, w, cut, 6000, BF16)


def test_product_leaves_other_rows_and_columns():
    """Rows of no group, and the columns between n and a wider output's stride, keep their values."""
    x, w, offsets, cut = product_inputs(1, [3, 0, 40], 70, 200, "e4m3", extra=9)
    buffer = torch.full((52, 100), 7.0, device="cuda")
    out = ops.mx_matmul(x, w, offsets, dtype=F32, out=buffer[:, 10:80])
    check_product(out, x, w, cut, 200, F32)
    assert (buffer[43:] == 7).all() and (buffer[:, :10] == 7).all() and (buffer[:, 80:] == 7).all()


def test_product_clamps_offsets():
    """Offsets past the rows, negative or falling never reach memory outside the matrices."""
    x, w, _, _ = product_inputs(2, [20], 64, 128, "e4m3")
    w = ops.MxTensor(w.data.expand(4, -1, -1).contiguous(), w.scales.expand(4, -1, -1).contiguous(), 128, "e2m1")
    for bad, cut in (([-5, 4, 10, 15, 2**30], [0, 4, 10, 15, 20]), ([0, 10, 5, 12, 20], [0, 10, 10, 12, 20]), ([30, 40, 50, 60, 70], [20] * 5),
                     ([3, 6, 6, 6, 6], [3, 6, 6, 6, 6]), ([-(2**31), 2**31 - 1, 0, 0, 0], [0, 20, 20, 20, 20])):
        buffer = torch.full((20, 64), 7.0, device="cuda")
        out = ops.mx_matmul(x, w, torch.tensor(bad, dtype=torch.int32, device="cuda"), dtype=F32, out=buffer)
        check_product(out, x, w, cut, 128, F32)
        assert (buffer[: cut[0]] == 7).all() and (buffer[cut[-1]:] == 7).all()


def test_product_extreme_scales():
    """Blocks far apart in size, sums past the largest f16 and f32, and blocks of zeros (scale byte 0)."""
    k = 256
    g = gen(9)
    xv = normal(g, 40, k)
    xv[:, 32:64] *= 2.0**60
    xv[:, 64:96] *= 2.0**-60
    xv[3] = 0
    xv[5, :128] = 0
    wv = normal(g, 1, 64, k)
    wv[:, :, 32:64] *= 2.0**-60
    wv[:, :, 64:96] *= 2.0**60
    wv[:, 7] = 0
    x, w = ops.mx_quantize(xv, "e4m3"), ops.mx_quantize(wv, "e2m1")
    check_product(ops.mx_matmul(x, w, dtype=F32), x, w, [0, 40], k, F32)
    assert (ops.mx_matmul(x, w, dtype=F32)[3] == 0).all()
    big, wbig = ops.mx_quantize(normal(g, 40, k) * 2.0**70, "e4m3"), ops.mx_quantize(normal(g, 1, 64, k) * 2.0**70, "e2m1")
    out = ops.mx_matmul(big, wbig, dtype=F32)
    want = ref.values(big.data, big.scales, k, "e4m3") @ ref.values(wbig.data, wbig.scales, k, "e2m1")[0].t()
    far = want.abs() > 2.0**130
    assert far.any() and not torch.isfinite(out[far]).any()


def test_product_nan_stays_in_its_row_and_column():
    x, w, offsets, cut = product_inputs(4, [30, 34], 80, 192, "e4m3")
    clean = ops.mx_matmul(x, w, offsets, dtype=F32)
    x.scales[10, 2] = 255
    x.data[50, 100] = 0x7F  # an E4M3 NaN
    w.scales[1, 20, 0] = 255
    out = ops.mx_matmul(x, w, offsets, dtype=F32)
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[10], nan[50], nan[30:, 20] = True, True, True
    assert torch.equal(torch.isnan(out), nan)
    same_bits(out[~nan], clean[~nan])


def test_product_same_every_time():
    x, w, offsets, _ = product_inputs(6, [5, 90, 0, 33, 1], 1000, 1408, "e4m3")
    first = ops.mx_matmul(x, w, offsets, dtype=F32)
    for _ in range(5):
        same_bits(ops.mx_matmul(x, w, offsets, dtype=F32), first)
    ops.sync()  # nothing gave up waiting


# ---------------------------------------------------------------- the residual norm


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype,ddtype", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16), (F32, None), (BF16, None)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (2, 128), (5, 1000), (4, 2048), (3, 2049), (2, 4096), (2, 6152), (1, 16384), (2, 40000), (700, 512)])
def test_add_rms_norm(rows, cols, dtype, ddtype, fmt):
    g = gen(rows + cols)
    hidden = (normal(g, rows, cols) * torch.exp2(3 * normal(g, rows, 1))).to(dtype)
    delta = None if ddtype is None else normal(g, rows, cols, dtype=ddtype)
    weight = 1 + 0.1 * normal(g, cols)
    before = hidden.clone()
    total, q, plain = ops.add_rms_norm(hidden, delta, weight, 1e-6, fmt=fmt, bf16=True)
    same_bits(hidden, before)
    want_sum = hidden if delta is None else (hidden.float() + delta.float()).to(dtype)
    same_bits(total, want_sum)
    x = total.double()
    norm = x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + 1e-6) * weight.double()
    # f32: the inverse, two products, each off by half a step
    off = (plain.double() - norm).abs()
    assert (off <= (half_step(BF16) + 4 * 2.0**-24) * norm.abs() * 1.001 + tiny(BF16)).all()
    # The codes hold the norm to half a step of theirs: a value of magnitude below twice its
    # block's largest power of two 2^p is off by at most half a step of 2^p, plus what is clamped
    # (7/6 or 480/448 of the largest value are cut to it).
    got = ref.values(q.data, q.scales, cols, fmt)
    blocks = -(-cols // 32)
    wide = torch.zeros(rows, blocks * 32, dtype=torch.float64, device="cuda")
    wide[:, :cols] = norm.abs()
    amax = wide.view(rows, blocks, 32).amax(dim=2)
    scale = q.scales[:, :blocks]
    # the scale byte is the exact norm's, or its neighbour's where the norm is within 4 2^-24 of a power of two
    lo = torch.frexp(amax * (1 - 2.0**-22)).exponent - 1
    hi = torch.frexp(amax * (1 + 2.0**-22)).exponent - 1
    e = scale.long() - 127 + (2 if fmt == "e2m1" else 8)
    live = amax > 2.0**-100
    assert (((e == lo) | (e == hi)) | ~live).all()
    step = ref.pow2(torch.where(live, e, torch.zeros_like(e))).repeat_interleave(32, 1)[:, :cols]
    tol = step / (2 if fmt == "e2m1" else 8)  # E2M1: half of 2^p is cut at most (8 to 6: 2^p/2); E4M3: 512 to 448: 2^p / 4
    tol = torch.where(norm.abs() > step * 1.5, step / 2 if fmt == "e2m1" else step / 4, tol)
    assert ((got - norm).abs() <= tol * 1.001).all()
    assert (q.scales[:, blocks:] == 0).all()
    # and they are exactly the quantisation of the f32 norm where bf16 holds it: through the bf16 output of the same call
    again = ops.add_rms_norm(hidden, delta, weight, 1e-6, fmt=fmt)
    assert again[2] is None and torch.equal(again[1].data, q.data) and torch.equal(again[1].scales, q.scales)


@pytest.mark.parametrize("dtype,ddtype", [(F32, BF16), (BF16, F32), (BF16, BF16), (BF16, None)])
@pytest.mark.parametrize("rows,cols", [(15000, 500), (7200, 1017), (3700, 2048), (1900, 4000), (1300, 6144), (1250, 5001), (1000, 8192), (800, 9999), (600, 16384)])
def test_add_rms_norm_many_rows(rows, cols, dtype, ddtype):
    """Rows that fill the GPU several times over, of every class of widths."""
    test_add_rms_norm(rows, cols, dtype, ddtype, "e4m3")


def test_add_rms_norm_in_place_and_special_rows():
    g = gen(2)
    hidden, delta, weight = normal(g, 4, 300), normal(g, 4, 300), normal(g, 300)
    hidden[1], delta[1] = 0, 0  # an empty (padded) row
    hidden[2, 7] = float("nan")
    want = ops.add_rms_norm(hidden, delta, weight, 1e-6, bf16=True)
    out, q, plain = ops.add_rms_norm(hidden, delta, weight, 1e-6, bf16=True, out=hidden)
    assert out.data_ptr() == hidden.data_ptr()
    same_bits(out, want[0])
    same_bits(plain, want[2])
    assert torch.equal(q.data, want[1].data) and torch.equal(q.scales, want[1].scales)
    assert (q.data[1] & 0x7F == 0).all() and (plain[1] == 0).all()
    assert (q.scales[2, :10] == 255).all() and torch.isnan(plain[2]).all()
    assert torch.isfinite(plain[[0, 1, 3]]).all()


# ---------------------------------------------------------------- tokens sorted by expert


def pairs(seed, tokens, k, experts, dropped=0.0):
    g = gen(seed)
    idx = torch.randint(0, experts, (tokens, k), generator=g, device="cuda", dtype=torch.int32)
    if dropped:
        idx[torch.rand(tokens, k, generator=g, device="cuda") < dropped] = -1
        idx[torch.rand(tokens, k, generator=g, device="cuda") < dropped / 4] = experts + 3
    return idx


PLANS = [(1, 1, 1, 0), (1, 6, 64, 0), (3, 2, 5, 0.5), (31, 1, 7, 0), (33, 6, 64, 0), (128, 8, 256, 0.2), (1000, 6, 64, 0.5), (700, 3, 1024, 0), (2500, 64, 8, 0.1),
         (40, 4, 3, 1.1)]


@pytest.mark.parametrize("tokens,k,experts,dropped", PLANS)
def test_sort_plan(tokens, k, experts, dropped):
    idx = pairs(tokens, tokens, k, experts, dropped)
    plan = ops.sort_plan(idx, experts)
    offsets, at = ref.sort_plan(idx.cpu(), experts)
    assert torch.equal(plan.offsets.cpu(), offsets) and torch.equal(plan.at.cpu(), at)


@pytest.mark.parametrize("value", [0, 5, -1, 8, 2**31 - 1, -(2**31)])
def test_sort_plan_one_value(value):
    """Every pair on one expert (the same index twice in a token too), or all dropped."""
    idx = torch.full((517, 3), value, dtype=torch.int32, device="cuda")
    plan = ops.sort_plan(idx, 8)
    offsets, at = ref.sort_plan(idx.cpu(), 8)
    assert torch.equal(plan.offsets.cpu(), offsets) and torch.equal(plan.at.cpu(), at)


def test_sort_plan_large():
    """A million pairs: against a stable sort."""
    idx = pairs(1, 150000, 7, 160, 0.3)
    plan = ops.sort_plan(idx, 160)
    flat = torch.where((idx >= 0) & (idx < 160), idx, torch.full_like(idx, 160)).reshape(-1)
    order = torch.argsort(flat, stable=True)
    at = torch.empty_like(flat)
    at[order] = torch.arange(flat.numel(), device="cuda", dtype=torch.int32)
    assert torch.equal(plan.at.reshape(-1), torch.where(flat < 160, at, torch.full_like(at, -1)))
    counts = torch.bincount(flat, minlength=161)[:160].cumsum(0)
    assert plan.offsets[0] == 0 and torch.equal(plan.offsets[1:].long(), counts)


def test_no_tokens():
    idx = torch.empty(0, 6, dtype=torch.int32, device="cuda")
    plan = ops.sort_plan(idx, 4)
    assert plan.offsets.tolist() == [0] * 5
    x = torch.empty(0, 64, device="cuda")
    assert ops.sort_rows(x, plan).shape == (0, 64)
    w = torch.empty(0, 6, device="cuda")
    assert ops.unsort_rows(x, plan, w).shape == (0, 64)
    gr, gw = ops.unsort_rows_backward(x, x, plan, w)
    assert gr.shape == (0, 64) and gw.shape == (0, 6)
    q = ops.mx_quantize(x, "e4m3")
    out = ops.mx_matmul(q, ops.mx_quantize(torch.randn(4, 32, 64, device="cuda"), "e2m1"), plan.offsets)
    assert out.shape == (0, 32) and ops.mx_dequantize(q).shape == (0, 64)
    assert ops.add_rms_norm(x, x, torch.ones(64, device="cuda"), 1e-6)[0].shape == (0, 64)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,k,experts,dropped,cols", [(1, 1, 1, 0, 1), (5, 2, 3, 0.4, 71), (33, 6, 64, 0.3, 256), (300, 6, 16, 0, 2048), (64, 16, 40, 0.5, 1000),
                                                            (20, 33, 8, 0.2, 96), (3, 8, 8, 0, 9000)])
def test_sort_and_back(tokens, k, experts, dropped, cols, dtype):
    g = gen(tokens + cols)
    idx = pairs(cols, tokens, k, experts, dropped)
    plan = ops.sort_plan(idx, experts)
    at = plan.at.long()
    live = at >= 0
    x = normal(g, tokens, cols, dtype=dtype)
    out = torch.full((tokens * k, cols), 7.0, dtype=dtype, device="cuda")
    rows = ops.sort_rows(x, plan, out=out)
    token = torch.arange(tokens, device="cuda").unsqueeze(1).expand(-1, k)
    kept = int(live.sum())
    want = torch.full_like(out, 7.0)
    want[at[live]] = x[token[live]]
    same_bits(rows, want)
    # back, with weights
    rows = normal(g, tokens * k, cols, dtype=dtype)
    weights = torch.rand(tokens, k, generator=g, device="cuda")
    v = torch.where(live.unsqueeze(2), rows[at.clamp(min=0)].double(), torch.zeros(1, dtype=torch.float64, device="cuda"))
    for wts, acc, out_dtype in ((weights, False, dtype), (None, False, dtype), (weights, True, F32), (weights, False, F32), (None, True, dtype)):
        terms = v * (1 if wts is None else wts.double().unsqueeze(2))
        base = normal(g, tokens, cols, dtype=out_dtype)
        y = ops.unsort_rows(rows, plan, wts, out=base.clone() if acc else None, dtype=out_dtype, accumulate=acc)
        total, size = terms.sum(dim=1), terms.abs().sum(dim=1)
        if acc:
            total, size = total + base.double(), size + base.double().abs()
        assert y.dtype == out_dtype
        assert ((y.double() - total).abs() <= (k + 1) * 2.0**-24 * size + half_step(out_dtype) * total.abs() * 1.001 + tiny(out_dtype)).all()
        if not acc:
            assert (y[~live.any(dim=1)] == 0).all()
    # the gradients
    gy = normal(g, tokens, cols, dtype=dtype)
    buffer = torch.full_like(rows, 7.0)
    gr, gw = ops.unsort_rows_backward(gy, rows, plan, weights, out=buffer)
    want = torch.full_like(rows, 7.0)
    want[at[live]] = (gy.float().unsqueeze(1) * weights.unsqueeze(2)).to(dtype)[live]
    same_bits(gr, want)
    dots = v * gy.double().unsqueeze(1)
    assert ((gw.double() - dots.sum(dim=2)).abs() <= cols * 2.0**-24 * dots.abs().sum(dim=2)).all() and (gw[~live] == 0).all()
    same_bits(ops.sort_rows_backward(rows, plan), ops.unsort_rows(rows, plan))
    # rows behind the kept ones are not read
    if kept < tokens * k:
        rows[kept:] = float("nan")
        assert torch.isfinite(ops.unsort_rows(rows, plan, weights)).all()
        assert torch.isfinite(ops.unsort_rows_backward(gy, rows, plan, weights)[1]).all()
    # in place
    clean = torch.where(torch.isnan(rows), torch.zeros_like(rows), rows)
    gr2, gw2 = ops.unsort_rows_backward(gy, clean, plan, weights, out=clean)
    same_bits(gr2[:kept], gr[:kept])
    same_bits(gw2, gw)


def test_gradients_against_differences():
    """<grad, d> of both directions against central differences of the f64 formula along d."""
    g = gen(11)
    tokens, k, experts, cols = 9, 4, 6, 48
    plan = ops.sort_plan(pairs(5, tokens, k, experts, 0.25), experts)
    at, live = plan.at.long(), plan.at >= 0
    x, rows, w = normal(g, tokens, cols), normal(g, tokens * k, cols), torch.rand(tokens, k, generator=g, device="cuda")
    gy, gs = normal(g, tokens, cols), normal(g, tokens * k, cols)

    def back(r, ww):
        return (torch.where(live.unsqueeze(2), r[at.clamp(min=0)], torch.zeros_like(r[:1])) * ww.unsqueeze(2)).sum(dim=1)

    def forth(xx):
        out = torch.zeros(tokens * k, cols, dtype=xx.dtype, device="cuda")
        out[at[live]] = xx.unsqueeze(1).expand(-1, k, -1)[live]
        return out

    gr, gw = ops.unsort_rows_backward(gy, rows, plan, w, out=torch.zeros_like(rows))
    gx = ops.sort_rows_backward(gs, plan)
    dr, dw, dx = (normal(g, *t.shape).double() for t in (rows, w, x))
    h = 1e-4
    for got, diff in (((gr.double() * dr).sum() + (gw.double() * dw).sum(),
                       ((back(rows.double() + h * dr, w.double() + h * dw) - back(rows.double() - h * dr, w.double() - h * dw)) * gy.double()).sum() / (2 * h)),
                      ((gx.double() * dx).sum(), ((forth(x.double() + h * dx) - forth(x.double() - h * dx)) * gs.double()).sum() / (2 * h))):
        # every product of the gradients is off by a few steps of f32; the formulas have no third derivative
        assert abs(float(got - diff)) <= 1e-4 * max(1.0, abs(float(diff)))


def test_sort_strides_types_and_mx_rows():
    g = gen(13)
    plan = ops.sort_plan(pairs(3, 40, 2, 8, 0.3), 8)
    at, live = plan.at.long(), plan.at >= 0
    token = torch.arange(40, device="cuda").unsqueeze(1).expand(-1, 2)
    kept = int(live.sum())
    wide = torch.randint(0, 100, (40, 90), generator=g, device="cuda")
    for x in (wide[:, 3:80].to(torch.uint8), wide.to(torch.uint8)[:, 3:80], wide.to(torch.int16)[:, 1:64], wide.int()[:, 1:50], wide.double()[:, 5:]):
        rows = ops.sort_rows(x, plan, out=torch.zeros(kept, x.shape[1], dtype=x.dtype, device="cuda"))
        want = torch.zeros_like(rows)
        want[at[live]] = x[token[live]]
        assert torch.equal(rows, want)
    buffer = torch.zeros(kept, 50, device="cuda")
    ops.sort_rows(wide[:, :20].float(), plan, out=buffer[:, 15:35])
    assert (buffer[:, :15] == 0).all() and (buffer[:, 35:] == 0).all()
    few = ops.sort_rows(wide.float(), plan, out=torch.zeros(5, 90, device="cuda"))  # room for five rows only
    assert torch.equal(few, ops.sort_rows(wide.float(), plan)[:5])
    q = ops.mx_quantize(normal(g, 40, 200), "e4m3")
    s = ops.sort_rows(q, plan)
    assert torch.equal(ops.mx_dequantize(s)[:kept][at[live]], ops.mx_dequantize(q)[token[live]])


# ---------------------------------------------------------------- together


def test_feed_forward_of_the_operators():
    """One expert layer as a runner composes it: residual norm, routing, sort, 4-bit products with
    SwiGLU between them, back with the weights, and the residual's next addition.  Each stage is
    checked in 64 bits on the stage before it."""
    g = gen(21)
    tokens, hidden, inter, experts, k = 53, 256, 160, 12, 3
    h, d, norm_w = normal(g, tokens, hidden), normal(g, tokens, hidden), 1 + 0.1 * normal(g, hidden)
    gate = ops.mx_quantize(normal(g, experts, inter, hidden, dtype=BF16) * 0.1, "e2m1")
    up = ops.mx_quantize(normal(g, experts, inter, hidden, dtype=BF16) * 0.1, "e2m1")
    down = ops.mx_quantize(normal(g, experts, hidden, inter, dtype=BF16) * 0.1, "e2m1")
    router = 0.1 * normal(g, experts, hidden)

    res, xq, xb = ops.add_rms_norm(h, d, norm_w, 1e-6, bf16=True)
    weights, idx = torch.topk(torch.softmax(xb.float() @ router.t(), dim=1), k, dim=1)
    idx, weights = idx.int().contiguous(), weights.contiguous()
    idx[5] = -1  # a padded token
    plan = ops.sort_plan(idx, experts)
    rows = ops.sort_rows(xq, plan)
    cut = plan.offsets.tolist()
    assert cut[-1] == (tokens - 1) * k
    a = ops.mx_matmul(rows, gate, plan.offsets, dtype=F32)
    b = ops.mx_matmul(rows, up, plan.offsets, dtype=F32)
    check_product(a, rows, gate, cut, hidden, F32)
    check_product(b, rows, up, cut, hidden, F32)
    act = torch.zeros(tokens * k, inter, device="cuda")
    from litemind_b200._lib import check, load

    check(load().lm_gemm_silu_multiply(a.data_ptr(), b.data_ptr(), act.data_ptr(), cut[-1] * inter, torch.cuda.current_stream().cuda_stream))
    hq = ops.mx_quantize(act, "e4m3")
    check_quantised(hq, act, "e4m3")
    y = ops.mx_matmul(hq, down, plan.offsets, dtype=BF16)
    check_product(y, hq, down, cut, inter, BF16)
    out = ops.unsort_rows(y, plan, weights, out=res.clone(), accumulate=True)
    live = plan.at >= 0
    terms = torch.where(live.unsqueeze(2), y[plan.at.long().clamp(min=0)].double(), torch.zeros(1, dtype=torch.float64, device="cuda")) * weights.double().unsqueeze(2)
    total = res.double() + terms.sum(dim=1)
    assert ((out.double() - total).abs() <= (k + 2) * 2.0**-24 * (res.double().abs() + terms.abs().sum(dim=1)) + tiny(F32)).all()
    same_bits(out[5], res[5])


def test_captured_and_replayed():
    """The whole chain in a CUDA graph on a side stream: new inputs in the same buffers, replayed twice."""
    g = gen(31)
    tokens, hidden, n, experts, k = 40, 512, 384, 8, 2
    h, d, w = normal(g, tokens, hidden), normal(g, tokens, hidden), 1 + 0.1 * normal(g, hidden)
    idx = pairs(4, tokens, k, experts, 0.2)
    weights = torch.rand(tokens, k, generator=g, device="cuda")
    wq = ops.mx_quantize(normal(g, experts, n, hidden), "e2m1")

    def chain(rows_buffer, y_buffer):
        res, q, _ = ops.add_rms_norm(h, d, w, 1e-6)
        plan = ops.sort_plan(idx, experts)
        rows = ops.sort_rows(q, plan, out=rows_buffer)
        y = ops.mx_matmul(rows, wq, plan.offsets, dtype=BF16, out=y_buffer)
        back = ops.unsort_rows(y, plan, weights, dtype=F32)
        gr, gw = ops.unsort_rows_backward(back.to(BF16), y, plan, weights, out=torch.zeros_like(y))
        return res, back, gr, gw, ops.sort_rows_backward(gr, plan)

    def buffers():
        r = ops.MxTensor.empty((tokens * k, hidden), "e4m3")
        r.data.zero_(), r.scales.zero_()
        return r, torch.zeros(tokens * k, n, dtype=BF16, device="cuda")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = buffers()
        chain(*mine)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = chain(*mine)
    for seed in (1, 2):
        gg = gen(seed)
        h.copy_(normal(gg, tokens, hidden))
        idx.copy_(pairs(seed, tokens, k, experts, 0.3))
        graph.replay()
        torch.cuda.synchronize()
        want = chain(*buffers())
        for a, b in zip(captured, want):
            same_bits(a, b)


def test_two_streams_at_once():
    """Products and sorts that overlap on two streams do not touch one another's results."""
    sets = [product_inputs(40 + i, [30, 7, 200, 0, 63], 1024, 2048, "e4m3") for i in range(2)]
    want = [ops.mx_matmul(x, w, o, dtype=F32) for x, w, o, _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, w, o, _ = sets[i]
                got[i].append(ops.mx_matmul(x, w, o, dtype=F32))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            same_bits(y, want[i])


FIRST_CALLS = """
import sys
sys.path.insert(0, {root!r})
import torch
from litemind_b200 import ops

torch.manual_seed(0)
x, d, w = torch.randn(300, 512, device="cuda"), torch.randn(300, 512, device="cuda"), torch.ones(512, device="cuda")
idx = torch.randint(0, 8, (1500, 2), device="cuda", dtype=torch.int32)
wide = torch.randn(1500, 512, device="cuda")
weights = torch.rand(1500, 2, device="cuda")
torch.cuda.synchronize()

def calls():
    total, q, plain = ops.add_rms_norm(x, d, w, 1e-6, bf16=True)
    m = ops.mx_quantize(x[:256], "e2m1")
    y = ops.mx_matmul(q, m, dtype=torch.float32)
    plan = ops.sort_plan(idx, 8)
    rows = ops.sort_rows(wide, plan)
    back = ops.unsort_rows(rows, plan, weights)
    gr, gw = ops.unsort_rows_backward(back, rows, plan, weights)
    return total, plain, ops.mx_dequantize(q), y, plan.offsets, plan.at, rows, back, gr, gw

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = calls()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(captured, calls()):
    assert torch.equal(a, b)
ops.sync()
print("equal")
"""


def test_first_calls_of_a_process_in_a_capture():
    """Nothing has to be called once before a capture."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=root)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "equal" in res.stdout, res.stdout + res.stderr


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_product_output_alignment(dtype):
    """Outputs that start on odd elements or have odd strides, every rest of a tile's columns."""
    for n in (64, 95, 96, 127, 128, 129):
        x, w, offsets, cut = product_inputs(n, [70, 0, 9], n, 160, "e4m3")
        for width, start in ((n, 0), (n + 1, 0), (n + 1, 1), (n + 2, 1), (n + 4, 2)):
            buffer = torch.full((79, width), 7.0, dtype=dtype, device="cuda")
            check_product(ops.mx_matmul(x, w, offsets, dtype=dtype, out=buffer[:, start:start + n]), x, w, cut, 160, dtype)
            assert (buffer[:, :start] == 7).all() and (buffer[:, start + n:] == 7).all()


def test_rows_past_32_bits():
    """Outputs and rows whose last elements lie past 2^31."""
    rows, n, k = 70000, 40000, 64
    x = ops.mx_quantize(normal(gen(1), rows, k, dtype=BF16), "e4m3")
    w = ops.mx_quantize(normal(gen(2), 1, n, k, dtype=BF16), "e2m1")
    out = ops.mx_matmul(x, w)
    tail = ops.MxTensor(x.data[-300:].contiguous(), x.scales[-300:].contiguous(), k, "e4m3")
    check_product(out[-300:], tail, w, [0, 300], k, BF16)
    del out
    n_rows, cols = 600000, 4096
    big = torch.zeros(n_rows, cols, dtype=BF16, device="cuda")
    at = torch.tensor([[n_rows - 1, 3], [n_rows - 2, -1], [n_rows - 5, 8]], dtype=torch.int32, device="cuda")
    plan = ops.SortPlan(torch.zeros(2, dtype=torch.int32, device="cuda"), at)
    v = normal(gen(3), 3, cols, dtype=BF16)
    ops.sort_rows(v, plan, out=big)
    for t, j, r in ((0, 0, n_rows - 1), (0, 1, 3), (1, 0, n_rows - 2), (2, 0, n_rows - 5), (2, 1, 8)):
        assert torch.equal(big[r], v[t])
    weights = torch.tensor([[1.0, 2.0], [4.0, 9.0], [0.5, 0.5]], device="cuda")
    y = ops.unsort_rows(big, plan, weights, dtype=F32)
    assert torch.equal(y, v.float() * torch.tensor([[3.0], [4.0], [1.0]], device="cuda"))
    gr, gw = ops.unsort_rows_backward(v, big, plan, weights, out=big)
    assert torch.equal(gr[n_rows - 2], v[1] * 4) and torch.equal(gr[8], v[2] * 0.5) and gw[1, 1] == 0


def test_other_streams_and_plans_at_once():
    """Plans of many pairs on two streams at once, and operators on a stream that is not the default."""
    sets = [pairs(50 + i, 4000, 6, 160, 0.2) for i in range(2)]
    want = [ref.sort_plan(s.cpu(), 160) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.sort_plan(sets[i], 160))
    torch.cuda.synchronize()
    for i in range(2):
        for plan in got[i]:
            assert torch.equal(plan.offsets.cpu(), want[i][0]) and torch.equal(plan.at.cpu(), want[i][1])


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_device():
    with torch.cuda.device(0):
        x = torch.randn(40, 256, device="cuda:1")
        q = ops.mx_quantize(x, "e4m3")
        w = ops.mx_quantize(torch.randn(64, 256, device="cuda:1"), "e2m1")
        y = ops.mx_matmul(q, w, dtype=F32)
        torch.cuda.synchronize(1)
        check_product(y, q, ops.MxTensor(w.data[None], w.scales[None], 256, "e2m1"), [0, 40], 256, F32)
        with pytest.raises(ValueError):
            ops.mx_matmul(q, ops.mx_quantize(torch.randn(64, 256, device="cuda:0"), "e2m1"))
