"""Calls of the stand-alone operators that their documentation allows, at the edges: experts that end
inside a warp, outputs in place of inputs, codes at the midpoints, gradients of other types, the
example that the documentation gives."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from litemind_b200 import _lib, ops  # noqa: E402
from tests import mx_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def same_bits(a, b):
    assert a.shape == b.shape and a.dtype == b.dtype
    kind = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    assert torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


@pytest.mark.parametrize("experts", [1, 7, 31, 33, 100, 255, 1000, 1023])
def test_sort_plan_over_a_cluster(experts):
    """More pairs than one CTA takes, experts that are no multiple of a warp."""
    idx = torch.randint(-1, experts + 1, (3001, 3), generator=gen(experts), device="cuda", dtype=torch.int32)
    plan = ops.sort_plan(idx, experts)
    offsets, at = ref.sort_plan(idx.cpu(), experts)
    assert torch.equal(plan.offsets.cpu(), offsets) and torch.equal(plan.at.cpu(), at)


def test_sort_rows_in_one_buffer():
    """Columns side by side, and rows behind one another, of one buffer are not the same memory."""
    plan = ops.sort_plan(torch.randint(0, 8, (40, 1), generator=gen(1), device="cuda", dtype=torch.int32), 8)
    for cols, strided in ((20, True), (64, True), (100, False)):
        buffer = normal(gen(cols), 80, 2 * cols)
        x = buffer[:40, :cols] if strided else buffer.view(-1)[: 40 * cols].view(40, cols)
        out = buffer[:40, cols:] if strided else buffer.view(-1)[40 * cols:80 * cols].view(40, cols)
        want = ops.sort_rows(x.clone(), plan)
        before = x.clone()
        same_bits(ops.sort_rows(x, plan, out=out), want)
        same_bits(x, before)
        even, odd = buffer[:80:2, :cols], buffer[1:80:2, 5:cols + 5]
        want = ops.sort_rows(even.clone(), plan)
        same_bits(ops.sort_rows(even, plan, out=odd), want)


def test_sort_rows_in_place_is_refused():
    plan = ops.sort_plan(torch.randint(0, 8, (40, 1), generator=gen(1), device="cuda", dtype=torch.int32), 8)
    buffer = normal(gen(2), 41, 64)
    before = buffer.clone()
    for x, out in ((buffer[:40], buffer[:40]), (buffer[:40], buffer[1:]), (buffer[:40, :32], buffer[:40, 31:63])):
        with pytest.raises(_lib.LiteMindError, match="overlaps x or at"):
            ops.sort_rows(x, plan, out=out)
    torch.cuda.synchronize()
    same_bits(buffer, before)


def test_mx_outputs_between_the_rows_of_inputs():
    """A buffer's columns as input and its other columns as output: not the same memory."""
    g = gen(3)
    buffer = normal(g, 64, 200, dtype=BF16)
    x = ops.mx_quantize(buffer[:, :96], "e4m3")
    w = ops.mx_quantize(normal(g, 100, 96), "e2m1")
    want = ops.mx_matmul(x, w)
    same_bits(ops.mx_matmul(x, w, out=buffer[:, 96:196]), want)
    same_bits(ops.mx_quantize(buffer[:, :96], "e4m3").data, x.data)
    few = ops.MxTensor(w.data[:64].contiguous(), w.scales[:64].contiguous(), 96, "e2m1")
    with pytest.raises(_lib.LiteMindError, match="overlaps an input"):
        ops.mx_matmul(x, few, out=x.data.view(BF16))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,k,experts,dropped,cols", [(1, 1, 1, 0, 1), (5, 2, 3, 0.4, 71), (33, 6, 64, 0.3, 256), (300, 6, 16, 0, 2048), (64, 16, 40, 0.5, 1000),
                                                            (20, 33, 8, 0.2, 96), (3, 8, 8, 0, 9000), (7, 3, 5, 1.1, 40)])
def test_gradient_of_an_f32_result(tokens, k, experts, dropped, cols, dtype):
    """grad_y in float32 with 16-bit rows: the products are rounded once, to the rows' type."""
    g = gen(tokens + cols)
    idx = torch.randint(0, experts, (tokens, k), generator=g, device="cuda", dtype=torch.int32)
    idx[torch.rand(tokens, k, generator=g, device="cuda") < dropped] = -1
    plan = ops.sort_plan(idx, experts)
    at, live = plan.at.long(), plan.at >= 0
    rows, gy = normal(g, tokens * k, cols, dtype=dtype), normal(g, tokens, cols)
    weights = torch.rand(tokens, k, generator=g, device="cuda")
    buffer = torch.full_like(rows, 7.0)
    gr, gw = ops.unsort_rows_backward(gy, rows, plan, weights, out=buffer)
    want = torch.full_like(rows, 7.0)
    want[at[live]] = (gy.unsqueeze(1) * weights.unsqueeze(2)).to(dtype)[live]
    same_bits(gr, want)
    v = torch.where(live.unsqueeze(2), rows[at.clamp(min=0)].double(), torch.zeros(1, dtype=torch.float64, device="cuda"))
    dots = v * gy.double().unsqueeze(1)
    # cols products added in f32: each addition is off by half a step, 2^-24, of at most the sum of magnitudes
    assert ((gw.double() - dots.sum(dim=2)).abs() <= cols * 2.0**-24 * dots.abs().sum(dim=2)).all() and (gw[~live] == 0).all()
    clean = rows.clone()
    gr2, gw2 = ops.unsort_rows_backward(gy, clean, plan, weights, out=clean)  # in place
    same_bits(gr2[at[live]], gr[at[live]])
    same_bits(gw2, gw)
    odd = torch.empty(tokens * cols + 1, device="cuda")[1:].view(tokens, cols).copy_(gy)  # no 16-byte boundary
    gr3, gw3 = ops.unsort_rows_backward(odd, rows, plan, weights, out=buffer.fill_(7.0))
    same_bits(gr3, want)
    assert ((gw3.double() - dots.sum(dim=2)).abs() <= cols * 2.0**-24 * dots.abs().sum(dim=2)).all()


def test_documented_chain():
    """The example of INTEGRATION.md as it stands there: it runs, and its gradients are the formulas'."""
    import os

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    part = text[text.index("## Operators on their own"):]
    part = part[: part.index("\n## ", 5)]
    blocks = [b.split("```")[0] for b in part.split("```python\n")[1:]]
    assert len(blocks) == 2
    g = gen(17)
    tokens, hidden, inter, experts, k = 29, 192, 96, 6, 2
    idx = torch.randint(-1, experts, (tokens, k), generator=g, device="cuda", dtype=torch.int32)
    names = dict(torch=torch, experts=experts, topk_idx=idx, topk_weights=torch.rand(tokens, k, generator=g, device="cuda"), hidden=normal(g, tokens, hidden),
                 delta=normal(g, tokens, hidden), norm_weight=1 + 0.1 * normal(g, hidden), gate_up=0.1 * normal(g, experts, 2 * inter, hidden),
                 down=0.1 * normal(g, experts, hidden, inter))
    exec(blocks[0], names)
    plan, y, delta = names["plan"], names["y"], names["delta"]
    assert delta.dtype == F32 and delta.shape == (tokens, hidden) and y.shape == (tokens * k, hidden)
    names.update(grad_delta=normal(g, tokens, hidden), grad_rows=normal(g, tokens * k, hidden))
    exec(blocks[1], names)
    at, live = plan.at.long().clamp(min=0), (plan.at >= 0).unsqueeze(2)
    zero = torch.zeros(1, dtype=torch.float64, device="cuda")
    dots = torch.where(live, y[at].double(), zero) * names["grad_delta"].double().unsqueeze(1)
    assert ((names["grad_weights"].double() - dots.sum(dim=2)).abs() <= hidden * 2.0**-24 * dots.abs().sum(dim=2)).all()
    want = names["grad_delta"].unsqueeze(1) * names["topk_weights"].unsqueeze(2)
    same_bits(names["grad_y"][at[live[..., 0]]], want.to(BF16)[live[..., 0]])
    terms = torch.where(live, names["grad_rows"][at].double(), zero)
    assert ((names["grad_x"].double() - terms.sum(dim=1)).abs() <= k * 2.0**-24 * terms.abs().sum(dim=1)).all()
    # and the result is the formula's on the stages before it
    terms = torch.where(live, y[at].double(), zero) * names["topk_weights"].double().unsqueeze(2)
    assert ((delta.double() - terms.sum(dim=1)).abs() <= (k + 1) * 2.0**-24 * terms.abs().sum(dim=1)).all()


def test_python_guards_behind_the_device_check():
    """The guards that CPU tensors never reach, each by its own message."""
    g = gen(5)
    x, w = ops.mx_quantize(normal(g, 4, 64), "e4m3"), ops.mx_quantize(normal(g, 3, 5, 64), "e2m1")
    offsets = torch.tensor([0, 1, 2, 4], device="cuda", dtype=torch.int32)
    plan = ops.SortPlan(torch.zeros(9, device="cuda", dtype=torch.int32), torch.zeros(4, 1, device="cuda", dtype=torch.int32))
    h, rows, weights, gain = normal(g, 4, 64), normal(g, 4, 64), torch.rand(4, 1, device="cuda"), torch.ones(64, device="cuda")
    out = torch.zeros(4, 5, dtype=BF16, device="cuda")
    cases = [(lambda: ops.mx_matmul(x, w), "several groups need offsets"), (lambda: ops.mx_matmul(x, w, offsets[:3]), "offsets must be int32"),
             (lambda: ops.mx_matmul(x, w, offsets.long()), "offsets must be int32"), (lambda: ops.mx_matmul(x, w, torch.stack((offsets, offsets), 1)[:, 0]), "offsets must be int32"),
             (lambda: ops.mx_matmul(x, w, offsets, out=out[:3]), "out has another shape or type"), (lambda: ops.mx_matmul(x, w, offsets, out=out.float()), "out has another shape or type"),
             (lambda: ops.mx_matmul(x, w, offsets, out=out[:1].expand(4, 5)), "out must be a matrix"),
             (lambda: ops.mx_matmul(x, w, offsets, dtype=torch.float64), "out must be float32, bfloat16"), (lambda: ops.mx_matmul(x, w, offsets.cpu()), "on one device"),
             (lambda: ops.mx_dequantize(x, BF16, out=torch.zeros(4, 64, device="cuda")), "out has another shape or type"),
             (lambda: ops.mx_dequantize(x, F32, out=torch.zeros(4, 65, device="cuda")[:, :64]), "not contiguous"), (lambda: ops.mx_dequantize(x, torch.float64), "out must be float32, bfloat16"),
             (lambda: ops.add_rms_norm(h, None, gain, 1e-6, out=h[:3]), "out must be contiguous"), (lambda: ops.add_rms_norm(h, None, gain, 1e-6, out=h.to(BF16)), "out must be contiguous"),
             (lambda: ops.add_rms_norm(h, None, gain.cpu(), 1e-6), "on one device"), (lambda: ops.unsort_rows_backward(h, rows, plan, weights, out=rows[:3]), "out must be contiguous"),
             (lambda: ops.unsort_rows_backward(h, rows, plan, weights, out=rows.to(BF16)), "out must be contiguous"), (lambda: ops.sort_rows(h.cpu(), plan), "on a CUDA device"),
             (lambda: ops.sort_rows(h, plan, out=rows.to(BF16)), "x's type and columns"), (lambda: ops.sort_rows(h, plan, out=rows[:, :63]), "x's type and columns"),
             (lambda: ops.unsort_rows(rows, plan, weights.cpu()), "on one device")]
    for n, (call, message) in enumerate(cases):
        with pytest.raises(ValueError, match=message):
            call()
            pytest.fail(f"case {n} was not refused")


# ---------------------------------------------------------------- the residual norm

# Every form of the kernel: one stretch of columns a thread, two (many bf16 rows), the sum read again
# (rows wider than 8192), rows that start on 16-byte words and rows that do not.
NORMS = [(3, 33), (5, 1000), (4, 2048), (3, 2049), (2, 6152), (1, 8200), (2, 40000), (15000, 500), (3700, 2048), (1250, 5001), (600, 16384), (400, 20001)]
TYPES = [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16), (BF16, None)]


def grid_index(a, fmt):
    """The index of the nearest of the format's magnitudes, ties to even, the largest for all beyond."""
    grid = (ref.E2M1 if fmt == "e2m1" else ref.E4M3).to(a.device)
    mid = (grid[1:] + grid[:-1]) / 2
    lo = torch.searchsorted(mid, a.contiguous())
    tie = (lo < mid.numel()) & (mid[lo.clamp(max=mid.numel() - 1)] == a)
    return torch.where(tie & (lo % 2 == 1), lo + 1, lo)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype,ddtype", TYPES)
@pytest.mark.parametrize("rows,cols", NORMS)
def test_norm_codes_are_the_nearest(rows, cols, dtype, ddtype, fmt):
    """The codes are the f64 norm's own, and a neighbour's only where the norm is within its f32 error
    of a midpoint: the inverse and two products are each off by half a step, 2^-24, 4 2^-24 in all with
    their second-order terms.  The scale likewise, at the powers of two."""
    g = gen(rows + cols)
    hidden = (normal(g, rows, cols) * torch.exp2(3 * normal(g, rows, 1))).to(dtype)
    delta = None if ddtype is None else normal(g, rows, cols, dtype=ddtype)
    weight = 1 + 0.1 * normal(g, cols)
    total, q, _ = ops.add_rms_norm(hidden, delta, weight, 1e-6, fmt=fmt)
    x = total.double()
    norm = x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + 1e-6) * weight.double()
    blocks, emax, by = -(-cols // 32), 2 if fmt == "e2m1" else 8, 4 * 2.0**-24
    wide = torch.zeros(rows, blocks * 32, dtype=torch.float64, device="cuda")
    wide[:, :cols] = norm
    amax = wide.view(rows, blocks, 32).abs().amax(dim=2)
    byte = q.scales[:, :blocks].long()

    def scale_of(a):
        return torch.where(a > 0, (torch.frexp(a).exponent.long() - 1 - emax + 127).clamp(min=0), torch.zeros_like(byte))

    assert ((byte >= scale_of(amax * (1 - by))) & (byte <= scale_of(amax * (1 + by)))).all()
    a = wide.abs() / ref.pow2(byte - 127).repeat_interleave(32, 1)
    if fmt == "e4m3":
        code = q.data[:, : blocks * 32].long()
    else:
        d = q.data[:, : blocks * 16].long()
        code = torch.stack((d % 16, d // 16), dim=-1).flatten(-2)
    sign_bit = 8 if fmt == "e2m1" else 128
    assert ((code % sign_bit >= grid_index(a * (1 - by), fmt)) & (code % sign_bit <= grid_index(a * (1 + by), fmt))).all()
    assert torch.equal(code >= sign_bit, torch.signbit(wide))
    assert (q.scales[:, blocks:] == 0).all() and (q.data[:, blocks * (32 if fmt == "e4m3" else 16):] == 0).all()


@pytest.mark.parametrize("dtype,ddtype", TYPES)
@pytest.mark.parametrize("rows,cols", NORMS)
def test_norm_in_place(rows, cols, dtype, ddtype):
    """The sum over hidden itself, and over delta where their types agree."""
    g = gen(rows + cols)
    hidden = normal(g, rows, cols, dtype=dtype)
    delta = None if ddtype is None else normal(g, rows, cols, dtype=ddtype)
    weight = 1 + 0.1 * normal(g, cols)
    want = ops.add_rms_norm(hidden, delta, weight, 1e-6, bf16=True)
    for over in ("hidden", "delta") if ddtype == dtype else ("hidden",):
        h, d = hidden.clone(), None if delta is None else delta.clone()
        total, q, plain = ops.add_rms_norm(h, d, weight, 1e-6, bf16=True, out=h if over == "hidden" else d)
        assert total is (h if over == "hidden" else d)
        same_bits(total, want[0])
        same_bits(plain, want[2])
        assert torch.equal(q.data, want[1].data) and torch.equal(q.scales, want[1].scales)
        if d is not None and over == "hidden":
            same_bits(d, delta)
        if over == "delta":
            same_bits(h, hidden)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(6, 33), (4, 2048), (2, 40000), (3700, 2048)])
@pytest.mark.parametrize("size", [2.0**127, 2.0**126 * 1.2, 2.0**-120, 2.0**-125, 2.0**-126])
def test_norm_at_the_ends_of_f32(size, rows, cols, dtype):
    """Rows near f32's largest and least normal numbers, epsilon 0: the norm is of ordinary size all the same."""
    g = gen(rows + cols)
    hidden = ((0.5 + 0.5 * torch.rand(rows, cols, generator=g, device="cuda")) * torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 0.5, -1.0, 1.0) * size).to(dtype)
    weight = 1 + 0.1 * normal(g, cols)
    _, _, plain = ops.add_rms_norm(hidden, None, weight, 0.0, bf16=True)
    x = hidden.double()
    norm = x / torch.sqrt((x * x).mean(dim=1, keepdim=True)) * weight.double()
    # bf16's half step and, in f32, the inverse (half of 2^-149 of 2^-128 at worst) and two products
    assert ((plain.double() - norm).abs() <= (2.0**-8 + 2.0**-22 + 2 * 2.0**-24) * norm.abs() * 1.001).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("power", [115, 100, -100, -118])
def test_norm_codes_at_the_ends_of_f32(power, fmt):
    """A power of two changes the norm of small whole numbers by nothing, as long as f32 holds the inverse."""
    hidden = torch.randint(-15, 16, (3, 512), generator=gen(2), device="cuda").float()
    weight = 1 + 0.1 * normal(gen(3), 512)
    want, got = (ops.add_rms_norm(hidden * s, None, weight, 0.0, fmt=fmt)[1] for s in (1.0, 2.0**power))
    assert torch.equal(got.data, want.data) and torch.equal(got.scales, want.scales)
