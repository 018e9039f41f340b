"""Cases of the microscaled expert path: MX quantisation and products, the residual norm with an
8-bit output, and tokens sorted by expert and back with their gradients.

Sizes are those of the DeepSeek-V2-Lite layer (hidden 2048, expert width 1408, 64 routed experts,
top-6, dense width 10944) and odd ones around them.  `run` has two forms: elementary torch
operations (own = False), or the calls of litemind_b200.ops (own = True).  Both take what `prepare`
makes: an MX matrix as the framework lays it out is
  data    uint8 [..., rows, pitch]   4-bit codes two a byte (the even column in the low half), or
                                     8-bit codes; columns padded with zeros to a multiple of 128
  scales  uint8 [..., rows, spitch]  one E8M0 byte for each 32 columns, padded to a multiple of 16
"""
import math
import random

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def up(n, m):
    return (n + m - 1) // m * m


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one token's activations on their way into an 8-bit product
        {"name": "quantise one row e4m3", "op": "quantise", "rows": 1, "cols": 2048, "dtype": "f32", "fmt": "e4m3"},
        # expert outputs of an odd width (no multiple of a block, a vector or a tile)
        {"name": "quantise odd rows e2m1", "op": "quantise", "rows": 1000, "cols": 1413, "dtype": "f32", "fmt": "e2m1"},
        # all gate projections of one layer, when a checkpoint's weights go to 4 bits
        {"name": "quantise expert weights e2m1", "op": "quantise", "rows": 90112, "cols": 2048, "dtype": "bf16", "fmt": "e2m1"},
        # one token's six experts, gate and up together: weights streamed for a single row each
        {"name": "product one token", "op": "product", "rows": 6, "groups": 64, "n": 2816, "k": 2048, "fmt": "e4m3", "out": "bf16", "skew": 0.0},
        # a decode batch of 128 tokens, every expert touched by a dozen rows
        {"name": "product decode 128", "op": "product", "rows": 768, "groups": 64, "n": 2816, "k": 2048, "fmt": "e4m3", "out": "bf16", "skew": 0.3},
        # a 4096-token prompt through the down projections, ragged loads, f32 for the combine
        {"name": "product prefill 4096", "op": "product", "rows": 24576, "groups": 64, "n": 2048, "k": 1408, "fmt": "e4m3", "out": "f32", "skew": 0.5},
        # the dense first layer's gate projection with both sides in 4 bits
        {"name": "product dense 4-bit", "op": "product", "rows": 4096, "groups": 1, "n": 10944, "k": 2048, "fmt": "e2m1", "out": "bf16", "skew": 0.0},
        # the norm before the experts for one decoded token, f32 residual as the runner keeps it
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 2048, "dtype": "f32", "delta": "f32", "router": True},
        # the same for a prompt, residual and update in bf16
        {"name": "norm prompt bf16", "op": "norm", "rows": 16384, "cols": 2048, "dtype": "bf16", "delta": "bf16", "router": False},
        # a small decode batch sorted by expert and brought back with its weights
        {"name": "sort decode 32", "op": "sort", "tokens": 32, "k": 6, "experts": 64, "local": 64, "hidden": 2048, "dtype": "bf16"},
        # a prompt on a rank that holds half of the experts: the other pairs are dropped
        {"name": "sort prompt half local", "op": "sort", "tokens": 16384, "k": 6, "experts": 64, "local": 32, "hidden": 2048, "dtype": "bf16"},
        # the gradients of both directions for a training batch
        {"name": "sort backward 8192", "op": "backward", "tokens": 8192, "k": 6, "experts": 64, "local": 64, "hidden": 2048, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantise", "product", "product", "norm", "sort", "backward"))
    if op == "quantise":
        return {"op": op, "rows": _log(rng, 1, 32768), "cols": _log(rng, 33, 5632), "dtype": rng.choice(("f32", "bf16", "f16")),
                "fmt": rng.choice(("e2m1", "e4m3"))}
    if op == "product":
        groups = rng.choice((1, 1, 8, 16, 64))
        n, k = _log(rng, 100, 2816), _log(rng, 100, 2816)
        return {"op": op, "rows": _log(rng, 1, 8192), "groups": groups, "n": n, "k": k, "fmt": rng.choice(("e4m3", "e4m3", "e2m1")),
                "out": rng.choice(("bf16", "f32", "f16")), "skew": rng.choice((0.0, 0.3, 0.6))}
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _log(rng, 64, 6144), "dtype": rng.choice(("f32", "bf16")),
                "delta": rng.choice(("f32", "bf16")), "router": rng.random() < 0.5}
    experts = rng.choice((8, 16, 64, 160))
    return {"op": op, "tokens": _log(rng, 1, 8192), "k": rng.randint(1, 8), "experts": experts,
            "local": rng.choice((experts, experts, experts // 2)), "hidden": _log(rng, 64, 2048), "dtype": rng.choice(("bf16", "bf16", "f32", "f16"))}


def counts(case):
    """Rows of each group, from the case alone: even when skew is 0, else log-normal shares."""
    g, r = case["groups"], case["rows"]
    rng = random.Random("%d %d %s" % (g, r, case["skew"]))
    if r < g:  # a few rows: one for each of some groups
        hit = set(rng.sample(range(g), r))
        return [int(i in hit) for i in range(g)]
    share = [math.exp(rng.gauss(0.0, case["skew"])) for _ in range(g)]
    total, at, cut = sum(share), 0.0, [0]
    for s in share:
        at += s
        cut.append(int(round(r * at / total)))
    cut[-1] = r
    return [b - a for a, b in zip(cut, cut[1:])]


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _row_scale(gen, rows):
    """Rows of activations differ in size by an order of magnitude or so."""
    return torch.exp2(torch.randn(rows, 1, generator=gen, device="cuda"))


def _outliers(x, gen):
    """A few channels of a residual stream are far larger than the rest."""
    cols = x.shape[1]
    at = torch.randint(0, cols, (max(1, cols // 256),), generator=gen, device="cuda")
    x[:, at] *= 24.0
    return x


def _pow2(e):
    """2^e in f32, for -126 <= e <= 127, from its bits: torch's own powers are rounded."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _block_scale(e):
    """2^e for a block's exponent, -127 (no normal number) among them."""
    return torch.where(e > -127, _pow2(e), torch.full_like(e, 2.0**-127, dtype=torch.float32))


def _pack(values, fmt):
    """An f32 matrix as data and scales in the framework's layout (as a checkpoint would hold it)."""
    rows, cols = values.shape
    wide = torch.zeros(rows, up(cols, 128), device=values.device)
    wide[:, :cols] = values
    codes, exps = _encode(wide, fmt)
    code = codes.to(torch.uint8)
    data = code if fmt == "e4m3" else code[:, 0::2] | (code[:, 1::2] << 4)
    blocks = (cols + 31) // 32
    scales = torch.zeros(rows, up(blocks, 16), dtype=torch.uint8, device=values.device)
    scales[:, :blocks] = (exps[:, :blocks] + 127).to(torch.uint8)
    return data.contiguous(), scales


def _encode(wide, fmt):
    """Codes (int32) and block exponents of an f32 matrix whose columns are a multiple of 32."""
    rows, cols = wide.shape
    b = wide.view(rows, cols // 32, 32)
    amax = b.abs().amax(dim=2)
    exps = torch.where(amax > 0, torch.frexp(amax).exponent - 1 - (2 if fmt == "e2m1" else 8), torch.full_like(amax, -127, dtype=torch.int32)).clamp_(-127, 127)
    v = (b * _pow2(-exps).unsqueeze(2)).view(rows, cols)
    a = v.abs()
    low, man, top = (0, 1, 6.0) if fmt == "e2m1" else (-6, 3, 448.0)
    e = (torch.frexp(a).exponent - 1).clamp_(min=low)
    q = (torch.round(a * _pow2(man - e)) * _pow2(e - man)).clamp_(max=top)
    e = torch.where(q > 0, (torch.frexp(q).exponent - 1).clamp_(min=low), torch.full_like(e, low))
    m = (q * _pow2(man - e)).to(torch.int32)  # 2^man + mantissa, or the mantissa alone below the least normal
    code = m + ((e - low) << man)
    return code + (torch.signbit(v).to(torch.int32) << (3 if fmt == "e2m1" else 7)), exps


def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    s = {"case": case}
    if op == "quantise":
        x = _normal(gen, case["rows"], case["cols"]) * (0.02 if case["rows"] > 20000 else 1.0)
        s["x"] = (x * _row_scale(gen, case["rows"])).to(DTYPES[case["dtype"]])
    elif op == "product":
        r, g, n, k = (case[c] for c in ("rows", "groups", "n", "k"))
        s["x"], s["xs"] = _pack(_normal(gen, r, k) * _row_scale(gen, r), case["fmt"])
        w = [_pack(_normal(gen, n, k) * 0.02, "e2m1") for _ in range(g)]
        s["w"], s["ws"] = torch.stack([a for a, _ in w]), torch.stack([b for _, b in w])
        c = counts(case)
        s["cap"] = max(c)
        hit = [i for i in range(g) if c[i]]
        s["hit"] = torch.tensor(hit, device="cuda") if len(hit) < g else None
        s["offsets"] = torch.tensor([0] + c, device="cuda").cumsum(0).to(torch.int32)
    elif op == "norm":
        x = _normal(gen, case["rows"], case["cols"]) * _row_scale(gen, case["rows"])
        s["hidden"] = _outliers(x, gen).to(DTYPES[case["dtype"]])
        s["delta"] = (0.25 * _normal(gen, case["rows"], case["cols"])).to(DTYPES[case["delta"]])
        s["weight"] = 1.0 + 0.1 * _normal(gen, case["cols"])
    else:
        t, k, e, h = (case[c] for c in ("tokens", "k", "experts", "hidden"))
        lean = 0.5 * _normal(gen, e)  # some experts are liked better
        score, idx = torch.topk(torch.softmax(_normal(gen, t, e) + lean, dim=1), k, dim=1)
        idx = idx.to(torch.int32)
        s["idx"] = torch.where(idx < case["local"], idx, torch.full_like(idx, -1))
        s["weights"] = score.contiguous()
        dt = DTYPES[case["dtype"]]
        flat = torch.where(s["idx"] >= 0, s["idx"], torch.full_like(idx, e)).reshape(-1)
        order = torch.argsort(flat, stable=True)
        s["kept"] = int((s["idx"] >= 0).sum())
        s["x"] = _normal(gen, t, h).to(dt)
        s["rows"] = _normal(gen, t * k, h).to(dt)  # what the experts gave back, in sorted order
        s["buffer"] = torch.zeros(t * k, h, dtype=dt, device="cuda")  # room for every pair; the dropped ones' rows stay as they are
        if op == "backward":
            s["offsets"] = torch.searchsorted(flat[order].contiguous(), torch.arange(case["local"] + 1, device="cuda", dtype=torch.int32)).to(torch.int32)
            at = torch.empty_like(flat)
            at[order] = torch.arange(t * k, device="cuda", dtype=torch.int32)
            s["at"] = torch.where(flat < e, at, torch.full_like(at, -1)).view(t, k)
            s["pairs"] = order[: s["kept"]]
            s["gy"] = _normal(gen, t, h).to(dt)
            s["grows"] = _normal(gen, t * k, h).to(dt)
    return s


# ---------------------------------------------------------------- the passes


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from litemind_b200 import ops

    case = s["case"]
    op = case["op"]
    if op == "quantise":
        q = ops.mx_quantize(s["x"], case["fmt"])
        return {"values": ops.mx_dequantize(q, torch.bfloat16), "scales": q.scales[:, : (case["cols"] + 31) // 32]}
    if op == "product":
        x = ops.MxTensor(s["x"], s["xs"], case["k"], case["fmt"])
        w = ops.MxTensor(s["w"], s["ws"], case["k"], "e2m1")
        return ops.mx_matmul(x, w, s["offsets"], dtype=DTYPES[case["out"]])
    if op == "norm":
        summed, q, plain = ops.add_rms_norm(s["hidden"], s["delta"], s["weight"], 1e-6, fmt="e4m3", bf16=case["router"])
        return {"hidden": summed, "values": ops.mx_dequantize(q, torch.bfloat16), "router": plain}
    if op == "sort":
        plan = ops.sort_plan(s["idx"], case["local"])
        rows = ops.sort_rows(s["x"], plan, out=s["buffer"])
        return {"offsets": plan.offsets, "at": plan.at, "rows": rows, "y": ops.unsort_rows(s["rows"], plan, s["weights"])}
    plan = ops.SortPlan(s["offsets"], s["at"])
    grows, gw = ops.unsort_rows_backward(s["gy"], s["rows"], plan, s["weights"], out=s["buffer"])
    return {"grad_rows": grows, "grad_weights": gw, "grad_x": ops.sort_rows_backward(s["grows"], plan)}


def _values(data, scales, cols, fmt):
    """What an MX matrix stands for, in f32."""
    if fmt == "e2m1":
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=data.device)
        v = torch.stack((table[(data & 15).int()], table[(data >> 4).int()]), dim=-1).flatten(-2)
    else:
        c = data.int()
        e, m = (c >> 3) & 15, c & 7
        v = torch.where(e > 0, m + 8, m).float() * _pow2(torch.clamp(e, min=1) - 10)
        v = torch.where(c > 127, -v, v)
    pad = v.shape[-1]
    e = scales[..., : pad // 32].int() - 127
    return (v.unflatten(-1, (pad // 32, 32)) * _block_scale(e).unsqueeze(-1)).flatten(-2)[..., :cols]


def _quantised(x, fmt):
    """The bf16 values that a matrix's MX form stands for, and its scale bytes."""
    rows, cols = x.shape
    wide = torch.zeros(rows, up(cols, 32), device=x.device)
    wide[:, :cols] = x.float()
    b = wide.view(rows, -1, 32)
    amax = b.abs().amax(dim=2, keepdim=True)
    top_e, low, man, top = (2, 0, 1, 6.0) if fmt == "e2m1" else (8, -6, 3, 448.0)
    exps = torch.where(amax > 0, torch.frexp(amax).exponent - 1 - top_e, torch.full_like(amax, -127, dtype=torch.int32)).clamp(-127, 127)
    v = b * _pow2(-exps)
    step = (torch.frexp(v).exponent - 1).clamp(min=low) - man
    q = (torch.round(v * _pow2(-step)) * _pow2(step)).clamp(-top, top)
    return (q * _block_scale(exps)).view(rows, -1)[:, :cols].to(torch.bfloat16), (exps + 127).squeeze(2).to(torch.uint8)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quantise":
        values, scales = _quantised(s["x"], case["fmt"])
        return {"values": values, "scales": scales}
    if op == "product":
        g, cap, r, k, n = case["groups"], s["cap"], case["rows"], case["k"], case["n"]
        x = _values(s["x"], s["xs"], k, case["fmt"])
        if g == 1:
            return (x @ _values(s["w"][0], s["ws"][0], k, "e2m1").t()).to(DTYPES[case["out"]])
        off, w, ws = s["offsets"].long(), s["w"], s["ws"]
        if s["hit"] is not None:  # groups without rows are not computed
            off, w, ws, g = torch.cat((off[s["hit"]], off[-1:])), w[s["hit"]], ws[s["hit"]], s["hit"].numel()
        row = torch.arange(r, device="cuda")
        group = torch.searchsorted(off[1:].contiguous(), row, right=True)
        slot = group * cap + row - off[group]
        padded = torch.zeros(g * cap, k, device="cuda")
        padded[slot] = x
        y = torch.bmm(padded.view(g, cap, k), _values(w, ws, k, "e2m1").transpose(1, 2))
        return y.view(g * cap, n)[slot].to(DTYPES[case["out"]])
    if op == "norm":
        summed = (s["hidden"].float() + s["delta"].float()).to(s["hidden"].dtype)
        x = summed.double()
        normed = (x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + 1e-6) * s["weight"].double()).float()
        return {"hidden": summed, "values": _quantised(normed, "e4m3")[0], "router": normed.to(torch.bfloat16) if case["router"] else None}
    if op == "sort":
        t, k, n = case["tokens"], case["k"], case["local"]
        flat = torch.where(s["idx"] >= 0, s["idx"], torch.full_like(s["idx"], n)).reshape(-1)
        order = torch.argsort(flat, stable=True)
        offsets = torch.bincount(flat, minlength=n + 1)[:n].cumsum(0)
        at = torch.empty_like(flat)
        at[order] = torch.arange(t * k, device="cuda", dtype=torch.int32)
        at = torch.where(flat < n, at, torch.full_like(at, -1)).view(t, k)
        rows = s["buffer"]
        rows[: s["kept"]] = s["x"][order[: s["kept"]] // k]
        w = torch.where(at >= 0, s["weights"], torch.zeros_like(s["weights"]))
        y = (s["rows"][at.clamp(min=0)].float() * w.unsqueeze(2)).sum(dim=1)
        return {"offsets": torch.cat((offsets.new_zeros(1), offsets)).to(torch.int32), "at": at, "rows": rows, "y": y.to(s["rows"].dtype)}
    at = s["at"]
    live, safe = at >= 0, at.clamp(min=0)
    gy, w = s["gy"].float(), s["weights"]
    pairs = s["pairs"]
    grad_rows = s["buffer"]
    grad_rows[: s["kept"]] = (gy[pairs // case["k"]] * w.reshape(-1)[pairs].unsqueeze(1)).to(grad_rows.dtype)
    grad_w = torch.where(live, (s["rows"][safe].float() * gy.unsqueeze(1)).sum(dim=2), torch.zeros_like(w))
    grad_x = torch.where(live.unsqueeze(2), s["grows"][safe].float(), torch.zeros(1, device="cuda")).sum(dim=1)
    return {"grad_rows": grad_rows, "grad_weights": grad_w, "grad_x": grad_x.to(s["gy"].dtype)}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "quantise":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * (SIZES[case["dtype"]] + 2) + r * ((c + 31) // 32), "flops": 4 * r * c}
    if op == "product":
        r, n, k = case["rows"], case["n"], case["k"]
        touched = sum(c > 0 for c in counts(case))
        blocks = (k + 31) // 32
        x = r * (k if case["fmt"] == "e4m3" else (k + 1) // 2) + r * blocks
        return {"bytes": x + touched * n * ((k + 1) // 2 + blocks) + r * n * SIZES[case["out"]], "flops": 2 * r * n * k}
    if op == "norm":
        r, c = case["rows"], case["cols"]
        per = 2 * SIZES[case["dtype"]] + SIZES[case["delta"]] + 2 + (2 if case["router"] else 0)
        return {"bytes": r * c * per + 4 * c, "flops": 8 * r * c}
    t, k, h, z = case["tokens"], case["k"], case["hidden"], SIZES[case["dtype"]]
    kept = t * k * case["local"] / case["experts"]
    if op == "sort":  # x once, its copies, the experts' rows, y; the pairs' indices and places
        return {"bytes": (2 * t + 2 * kept) * h * z + 12 * t * k, "flops": 2 * kept * h}
    return {"bytes": (2 * t + 3 * kept) * h * z + 12 * t * k, "flops": 4 * kept * h}


# ---------------------------------------------------------------- the definition in 64 bits


def _exact_pow2(e):
    """2^e in f64 for a whole number e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_values(data, scales, cols, fmt):
    d = data.long()
    if fmt == "e2m1":
        d = torch.stack((d % 16, d // 16), dim=-1).reshape(*d.shape[:-1], -1)
    bits, man, bias = (4, 1, 1) if fmt == "e2m1" else (8, 3, 7)
    sign = 1.0 - 2.0 * (d >= 2 ** (bits - 1)).double()
    mag = d % 2 ** (bits - 1)
    field, frac = mag // 2**man, (mag % 2**man).double() / 2**man
    v = torch.where(field == 0, frac * 2.0 ** (1 - bias), (1.0 + frac) * _exact_pow2(field - bias))
    f = _exact_pow2(scales.long() - 127).repeat_interleave(32, dim=-1)
    return (sign * v * f[..., : v.shape[-1]])[..., :cols]


def _exact_mx(x, fmt):
    """Each block's scale from its largest value, then the nearest of the format's values (even on ties)."""
    rows, cols = x.shape
    if fmt == "e2m1":
        grid = torch.tensor(E2M1, dtype=torch.float64)
    else:
        grid = torch.tensor([m / 8 * 2.0**-6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1], dtype=torch.float64)
    grid = grid.cuda()
    mid = (grid[1:] + grid[:-1]) / 2
    wide = torch.zeros(rows, up(cols, 32), dtype=torch.float64, device="cuda")
    wide[:, :cols] = x
    b = wide.view(rows, -1, 32)
    amax = b.abs().amax(dim=2, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent.long() - 1 - (2 if fmt == "e2m1" else 8), torch.full_like(amax, -127, dtype=torch.long)).clamp(-127, 127)
    a = b.abs() / _exact_pow2(e)
    lo = torch.searchsorted(mid, a.contiguous())  # the first midpoint that is not below
    tie = (lo < mid.numel()) & (mid[lo.clamp(max=mid.numel() - 1)] == a)
    at = torch.where(tie & (lo % 2 == 1), lo + 1, lo)
    return (torch.sign(b) * grid[at] * _exact_pow2(e)).view(rows, -1)[:, :cols], (e + 127).squeeze(2).to(torch.uint8)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantise":
        values, scales = _exact_mx(s["x"].double(), case["fmt"])
        return {"values": values, "scales": scales}
    if op == "product":
        x = _exact_values(s["x"], s["xs"], case["k"], case["fmt"])
        cut = s["offsets"].tolist()
        return torch.cat([x[a:b] @ _exact_values(s["w"][g], s["ws"][g], case["k"], "e2m1").t() for g, (a, b) in enumerate(zip(cut, cut[1:])) if b > a])
    if op == "norm":
        summed = s["hidden"].double() + s["delta"].double()
        x = summed.float().to(s["hidden"].dtype).double()  # the stored residual is what is normalised
        normed = x / torch.sqrt((x * x).sum(dim=1, keepdim=True) / case["cols"] + 1e-6) * s["weight"].double()
        return {"hidden": summed, "values": _exact_mx(normed, "e4m3")[0], "router": normed if case["router"] else None}
    idx, t, k = s["idx"].reshape(-1), case["tokens"], case["k"]
    pairs = torch.cat([torch.nonzero(idx == e).flatten() for e in range(case["local"])])
    token, row = pairs // k, torch.arange(pairs.numel(), device="cuda")
    w = s["weights"].reshape(-1).double()[pairs].unsqueeze(1)

    def back(v):
        return torch.zeros(t, case["hidden"], dtype=torch.float64, device="cuda").index_add_(0, token, v)

    def padded(v):
        return torch.cat((v, v.new_zeros(t * k - v.shape[0], v.shape[1])))

    if op == "sort":
        return {"offsets": None, "at": None, "rows": padded(s["x"].double()[token]), "y": back(s["rows"].double()[row] * w)}
    gy = s["gy"].double()[token]
    gw = torch.zeros(t * k, dtype=torch.float64, device="cuda")
    gw[pairs] = (gy * s["rows"].double()[row]).sum(dim=1)
    return {"grad_rows": padded(gy * w), "grad_weights": gw.view(t, k), "grad_x": back(s["grows"].double()[row])}
