"""The stand-alone operators of the C ABI on torch tensors: MX matrices (quantise, dequantise,
grouped product), the residual's addition and RMS norm with an MX output, and tokens sorted by
expert and back with their gradients.

As in ``moe.py`` torch is the device-memory plumbing and all arithmetic runs in
liblitemind_b200.so on the GPU.  Every call works on its tensors' device and that device's current
stream, allocates its outputs with torch unless it is given them, and raises ``ValueError`` for an
argument that does not fit (before any launch) or ``LiteMindError`` with the library's message.
"""
from __future__ import annotations

from contextlib import nullcontext

import torch

from . import _lib
from ._lib import check, load

_DTYPES = {torch.float32: _lib.LM_DTYPE_F32, torch.bfloat16: _lib.LM_DTYPE_BF16, torch.float16: _lib.LM_DTYPE_F16}
_FORMATS = {"e2m1": _lib.LM_MX_E2M1, "e4m3": _lib.LM_MX_E4M3}


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _same_device(*tensors) -> torch.device:
    """The one CUDA device that all the tensors (None left out) are on."""
    device = None
    for t in tensors:
        if t is not None:
            _need(t.is_cuda, "tensors must be on a CUDA device")
            if device is None:
                device = t.device
            else:
                _need(t.device == device, "all tensors must be on one device")
    return device


def _on(device: torch.device):
    """Makes `device` current for a call, when it is not."""
    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _matrix(t, name: str):
    _need(t.dim() == 2 and (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]),
          f"{name} must be a matrix with contiguous, non-overlapping rows")


def _row_stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _dtype(t, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    _need(code is not None, f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _format(fmt: str) -> int:
    code = _FORMATS.get(fmt)
    _need(code is not None, f"unknown MX format {fmt!r}: e2m1 or e4m3")
    return code


# ---------------------------------------------------------------- MX matrices


def _pad(n: int, to: int) -> int:
    return -(-n // to) * to


class MxTensor:
    """An MX matrix, or a stack of them, in the layout of include/litemind_moe.h.

    data    uint8 [..., rows, pitch]: 4-bit codes two a byte (``fmt`` "e2m1") or 8-bit codes ("e4m3"),
            padded with zeros to a multiple of 128 columns
    scales  uint8 [..., rows, pitch]: an E8M0 byte for each 32 columns, padded with zeros to a multiple of 16
    cols    columns of the matrix without the padding
    """

    __slots__ = ("data", "scales", "cols", "fmt")

    def __init__(self, data, scales, cols: int, fmt: str):
        _format(fmt)
        _need(data.dtype == torch.uint8 and scales.dtype == torch.uint8 and data.is_contiguous() and scales.is_contiguous(),
              "data and scales must be contiguous uint8 tensors")
        wide = _pad(cols, 128)
        _need(data.dim() >= 2 and data.shape[:-1] == scales.shape[:-1] and data.shape[-1] == (wide // 2 if fmt == "e2m1" else wide)
              and scales.shape[-1] == _pad(cols, 512) // 32, f"data and scales do not have the layout of {cols} {fmt} columns")
        self.data, self.scales, self.cols, self.fmt = data, scales, cols, fmt

    @classmethod
    def empty(cls, shape, fmt: str, device="cuda") -> "MxTensor":
        """An uninitialised one of the given [..., rows, cols]."""
        *lead, cols = shape
        wide = _pad(cols, 128)
        return cls(torch.empty((*lead, wide // 2 if fmt == "e2m1" else wide), dtype=torch.uint8, device=device),
                   torch.empty((*lead, _pad(cols, 512) // 32), dtype=torch.uint8, device=device), cols, fmt)

    @property
    def shape(self) -> tuple:
        return (*self.data.shape[:-1], self.cols)

    @property
    def rows(self) -> int:
        """Rows of all matrices of the stack together."""
        n = 1
        for d in self.data.shape[:-1]:
            n *= d
        return n


def mx_quantize(values, fmt: str, out: MxTensor | None = None) -> MxTensor:
    """lm_mx_quantize of a float32, bfloat16 or float16 [..., cols] tensor (more than two
    dimensions: contiguous)."""
    code = _dtype(values, "values")
    if values.dim() == 2:
        _matrix(values, "values")
        flat = values
    else:
        _need(values.dim() > 2 and values.is_contiguous(), "values must be a matrix, or contiguous with more dimensions")
        flat = values.view(-1, values.shape[-1])
    device = _same_device(values)
    if out is None:
        out = MxTensor.empty(values.shape, fmt, device)
    else:
        _need(out.shape == tuple(values.shape) and out.fmt == fmt, "out has another shape or format")
        _same_device(values, out.data, out.scales)
    with _on(device):
        check(load().lm_mx_quantize(flat.data_ptr(), code, flat.shape[0], flat.shape[1], _row_stride(flat), _format(fmt),
                                    out.data.data_ptr(), out.scales.data_ptr(), _stream(device)))
    return out


def mx_dequantize(x: MxTensor, dtype=torch.float32, out=None):
    """lm_mx_dequantize: the values that x stands for, as `dtype`."""
    device = _same_device(x.data, x.scales)
    if out is None:
        out = torch.empty(x.shape, dtype=dtype, device=device)
    else:
        _need(tuple(out.shape) == x.shape and out.dtype == dtype and out.is_contiguous(), "out has another shape or type, or is not contiguous")
        _same_device(x.data, out)
    code = _dtype(out, "out")
    with _on(device):
        check(load().lm_mx_dequantize(x.data.data_ptr(), x.scales.data_ptr(), _FORMATS[x.fmt], x.rows, x.cols, out.data_ptr(), code, x.cols,
                                      _stream(device)))
    return out


def mx_matmul(x: MxTensor, w: MxTensor, offsets=None, dtype=torch.bfloat16, out=None):
    """lm_mx_matmul: x [rows, k], sorted by group, times the transposed 4-bit w [groups, n, k] of
    each row's group -> [rows, n] of `dtype`.

    offsets: int32 [groups + 1] on the device (SortPlan.offsets); None with one group (w may be
    [n, k] then).  Rows of no group keep what `out` held."""
    _need(x.data.dim() == 2 and w.data.dim() in (2, 3) and w.fmt == "e2m1" and x.cols == w.cols,
          "x must be [rows, k] and w 4-bit [groups, n, k] with the same k")
    groups = w.data.shape[0] if w.data.dim() == 3 else 1
    rows, n = x.data.shape[0], w.data.shape[-2]
    device = _same_device(x.data, x.scales, w.data, w.scales, offsets, out)
    if offsets is None:
        _need(groups == 1, "several groups need offsets")
    else:
        _need(offsets.dtype == torch.int32 and offsets.is_contiguous() and offsets.numel() == groups + 1, "offsets must be int32 [groups + 1]")
    if out is None:
        out = torch.empty((rows, n), dtype=dtype, device=device)
    else:
        _need(tuple(out.shape) == (rows, n) and out.dtype == dtype, "out has another shape or type")
        _matrix(out, "out")
    code = _dtype(out, "out")
    with _on(device):
        check(load().lm_mx_matmul(x.data.data_ptr(), x.scales.data_ptr(), _FORMATS[x.fmt], rows, w.data.data_ptr(), w.scales.data_ptr(), groups, n,
                                  x.cols, None if offsets is None else offsets.data_ptr(), out.data_ptr(), code, _row_stride(out), _stream(device)))
    return out


def sync(device=None) -> None:
    """lm_ops_sync: waits for the device's current stream and raises if a kernel gave up waiting."""
    device = torch.device("cuda", torch.cuda.current_device() if device is None else torch.device(device).index or 0)
    with _on(device):
        check(load().lm_ops_sync(_stream(device)))


def add_rms_norm(hidden, delta, weight, eps: float, fmt: str = "e4m3", bf16: bool = False, out=None):
    """lm_gemm_add_rms_norm_mx: (hidden + delta, its RMS norm as an MxTensor, the norm in bfloat16
    or None).  hidden and delta (may be None): contiguous float32 or bfloat16 [rows, cols]; weight
    float32 [cols].  The sum has hidden's type and goes to `out`, which may be hidden itself."""
    _need(hidden.dim() == 2 and hidden.is_contiguous() and hidden.dtype in (torch.float32, torch.bfloat16), "hidden must be contiguous float32 or bfloat16 [rows, cols]")
    if delta is not None:
        _need(delta.shape == hidden.shape and delta.is_contiguous() and delta.dtype in (torch.float32, torch.bfloat16),
              "delta must be contiguous float32 or bfloat16 of hidden's shape")
    rows, cols = hidden.shape
    _need(weight.dtype == torch.float32 and weight.is_contiguous() and tuple(weight.shape) == (cols,), "weight must be contiguous float32 [cols]")
    device = _same_device(hidden, delta, weight, out)
    if out is None:
        out = torch.empty_like(hidden)
    else:
        _need(out.shape == hidden.shape and out.dtype == hidden.dtype and out.is_contiguous(), "out must be contiguous, of hidden's shape and type")
    q = MxTensor.empty((rows, cols), fmt, device)
    plain = torch.empty((rows, cols), dtype=torch.bfloat16, device=device) if bf16 else None
    with _on(device):
        check(load().lm_gemm_add_rms_norm_mx(hidden.data_ptr(), _DTYPES[hidden.dtype], None if delta is None else delta.data_ptr(),
                                             _DTYPES[hidden.dtype if delta is None else delta.dtype], weight.data_ptr(), rows, cols, eps,
                                             out.data_ptr(), None if plain is None else plain.data_ptr(), _FORMATS[fmt], q.data.data_ptr(),
                                             q.scales.data_ptr(), _stream(device)))
    return out, q, plain


# ---------------------------------------------------------------- tokens sorted by expert


class SortPlan:
    """Where each (token, slot) pair's row is among the rows sorted by expert (lm_moe_sort_plan).

    offsets  int32 [experts + 1]: expert e's rows are offsets[e] .. offsets[e + 1] - 1
    at       int32 [tokens, top_k]: the pair's row, -1 when dropped
    """

    __slots__ = ("offsets", "at")

    def __init__(self, offsets, at):
        _need(offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.is_contiguous() and at.dtype == torch.int32 and at.dim() == 2
              and at.is_contiguous(), "offsets must be int32 [experts + 1] and at int32 [tokens, top_k], contiguous")
        self.offsets, self.at = offsets, at


def sort_plan(topk_idx, experts: int) -> SortPlan:
    """lm_moe_sort_plan of int32 [tokens, top_k] expert indices (outside [0, experts): dropped)."""
    _need(topk_idx.dtype == torch.int32 and topk_idx.dim() == 2 and topk_idx.is_contiguous(), "topk_idx must be contiguous int32 [tokens, top_k]")
    _need(0 < experts <= 1024, "experts must be in 1 .. 1024")
    device = _same_device(topk_idx)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=device)
    at = torch.empty_like(topk_idx)
    with _on(device):
        check(load().lm_moe_sort_plan(topk_idx.data_ptr(), topk_idx.shape[0], topk_idx.shape[1], experts, offsets.data_ptr(), at.data_ptr(),
                                      _stream(device)))
    return SortPlan(offsets, at)


def _sort(x, plan: SortPlan, out):
    _matrix(x, "x")
    tokens, k = plan.at.shape
    _need(x.shape[0] == tokens, "x must have a row for each token of the plan")
    if out is None:
        out = torch.empty((tokens * k, x.shape[1]), dtype=x.dtype, device=x.device)
    else:
        _matrix(out, "out")
        _need(out.dtype == x.dtype and out.shape[1] == x.shape[1], "out must have x's type and columns")
    device = _same_device(x, plan.at, out)
    z = x.element_size()
    with _on(device):
        check(load().lm_moe_sort_rows(x.data_ptr(), _row_stride(x) * z, plan.at.data_ptr(), tokens, k, x.shape[1] * z, out.data_ptr(),
                                      _row_stride(out) * z, out.shape[0], _stream(device)))
    return out


def sort_rows(x, plan: SortPlan, out=None):
    """lm_moe_sort_rows: x [tokens, cols] (any type, or an MxTensor) -> its rows sorted by expert,
    one for each kept pair.  Rows behind the last kept pair keep what `out` held (uninitialised
    without it); `out` may have fewer rows than tokens * top_k when pairs are dropped."""
    if isinstance(x, MxTensor):
        _need(out is None or (out.fmt == x.fmt and out.cols == x.cols), "out must have x's format and columns")
        return MxTensor(_sort(x.data, plan, None if out is None else out.data), _sort(x.scales, plan, None if out is None else out.scales), x.cols, x.fmt)
    return _sort(x, plan, out)


def unsort_rows(rows, plan: SortPlan, weights=None, out=None, dtype=None, accumulate: bool = False):
    """lm_moe_unsort_rows: y[t] = sum_j weights[t, j] rows[at[t, j]] -> [tokens, cols] of `dtype`
    (rows' type by default, or float32).  weights: float32 [tokens, top_k], None for 1.
    accumulate adds to `out`."""
    _need(rows.dim() == 2 and rows.is_contiguous(), "rows must be a contiguous matrix")
    code = _dtype(rows, "rows")
    tokens, k = plan.at.shape
    if weights is not None:
        _need(weights.dtype == torch.float32 and weights.shape == plan.at.shape and weights.is_contiguous(), "weights must be contiguous float32 [tokens, top_k]")
    if out is None:
        _need(not accumulate, "accumulate needs out")
        out = torch.empty((tokens, rows.shape[1]), dtype=dtype or rows.dtype, device=rows.device)
    else:
        _need(tuple(out.shape) == (tokens, rows.shape[1]) and out.is_contiguous() and (dtype is None or out.dtype == dtype),
              "out must be contiguous [tokens, cols] of the given type")
    _need(out.dtype in (rows.dtype, torch.float32), "the result has rows' type or float32")
    device = _same_device(rows, plan.at, weights, out)
    with _on(device):
        check(load().lm_moe_unsort_rows(rows.data_ptr(), code, rows.shape[0], plan.at.data_ptr(), None if weights is None else weights.data_ptr(), tokens, k,
                                        rows.shape[1], out.data_ptr(), _DTYPES[out.dtype], int(accumulate), _stream(device)))
    return out


def sort_rows_backward(grad_rows, plan: SortPlan, out=None, dtype=None):
    """The gradient of sort_rows: grad_x[t] = sum_j grad_rows[at[t, j]]."""
    return unsort_rows(grad_rows, plan, None, out, dtype)


def unsort_rows_backward(grad_y, rows, plan: SortPlan, weights, out=None):
    """lm_moe_unsort_rows_backward: (grad_rows, grad_weights) of unsort_rows with weights.
    grad_rows goes to `out` (which may be rows itself); rows of no pair keep what it held
    (uninitialised without it)."""
    _need(rows.dim() == 2 and rows.is_contiguous() and grad_y.dim() == 2 and grad_y.is_contiguous() and grad_y.dtype == rows.dtype,
          "grad_y and rows must be contiguous matrices of one type")
    code = _dtype(rows, "rows")
    tokens, k = plan.at.shape
    _need(tuple(grad_y.shape) == (tokens, rows.shape[1]), "grad_y must be [tokens, cols]")
    _need(weights.dtype == torch.float32 and weights.shape == plan.at.shape and weights.is_contiguous(), "weights must be contiguous float32 [tokens, top_k]")
    if out is None:
        out = torch.empty_like(rows)
    else:
        _need(out.shape == rows.shape and out.dtype == rows.dtype and out.is_contiguous(), "out must be contiguous, of rows' shape and type")
    device = _same_device(grad_y, rows, plan.at, weights, out)
    grad_weights = torch.empty_like(weights)
    with _on(device):
        check(load().lm_moe_unsort_rows_backward(grad_y.data_ptr(), rows.data_ptr(), code, rows.shape[0], plan.at.data_ptr(), weights.data_ptr(), tokens, k,
                                                 rows.shape[1], out.data_ptr(), grad_weights.data_ptr(), _stream(device)))
    return out, grad_weights
