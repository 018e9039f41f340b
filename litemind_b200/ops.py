"""The stand-alone operators of the C ABI on torch tensors: MX matrices (quantise, dequantise,
grouped product), the residual's addition and RMS norm with an MX output, and tokens sorted by
expert and back with their gradients.

As in ``moe.py`` torch is the device-memory plumbing and all arithmetic runs in
liblitemind_b200.so on the GPU.  Every call works on its tensors' device and that device's current
stream, allocates its outputs with torch unless it is given them, and raises ``ValueError`` for an
argument that does not fit (before any launch) or ``LiteMindError`` with the library's message.
No autograd graph is recorded: the gradients are calls of their own.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check, load

_DTYPES = {torch.float32: _lib.LM_DTYPE_F32, torch.bfloat16: _lib.LM_DTYPE_BF16, torch.float16: _lib.LM_DTYPE_F16}
_FORMATS = {"e2m1": _lib.LM_MX_E2M1, "e4m3": _lib.LM_MX_E4M3}
_RESIDUAL = (torch.float32, torch.bfloat16)

# The calls for a few rows take a few microseconds on the GPU, so what Python adds counts: messages
# are made only when they are raised, outputs with new_empty (cheaper than torch.empty with a
# device), and the stream's handle is taken without building a torch.cuda.Stream (2 us).
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _index(first, *others) -> int:
    """The index of the one CUDA device that all the tensors (None left out) are on."""
    index = first.get_device()
    if index < 0:
        raise ValueError("tensors must be on a CUDA device")
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError("all tensors must be on one device")
    return index


def _call(fn, index: int, *args) -> None:
    """fn(*args, stream) with the device current and its current stream."""
    if torch.cuda.current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        check(status)


def _row_stride(t, name: str) -> int:
    """Elements from row to row of a matrix with contiguous rows that do not overlap."""
    if t.dim() == 2:
        rows, cols = t.shape
        if rows <= 1 or cols == 0:
            stride = cols
        else:
            stride = t.stride(0)
        if (cols <= 1 or t.stride(1) == 1) and stride >= cols:
            return stride
    raise ValueError(f"{name} must be a matrix with contiguous, non-overlapping rows")


def _dtype(t, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _format(fmt: str) -> int:
    code = _FORMATS.get(fmt)
    if code is None:
        raise ValueError(f"unknown MX format {fmt!r}: e2m1 or e4m3")
    return code


def _full(t, shape, dtype, message: str) -> None:
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(message)


# ---------------------------------------------------------------- MX matrices


def _pitches(cols: int, fmt: str) -> tuple:
    """Bytes of one row of data and of scales (lm_mx_data_pitch, lm_mx_scale_pitch)."""
    wide = -(-cols // 128) * 128
    return (wide // 2 if fmt == "e2m1" else wide), -(-cols // 512) * 16


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
        if data.dim() < 2 or data.shape[:-1] != scales.shape[:-1] or (data.shape[-1], scales.shape[-1]) != _pitches(cols, fmt):
            raise ValueError(f"data and scales do not have the layout of {cols} {fmt} columns")
        self.data, self.scales, self.cols, self.fmt = data, scales, cols, fmt

    @classmethod
    def empty(cls, shape, fmt: str, device="cuda") -> "MxTensor":
        """An uninitialised one of the given [..., rows, cols]."""
        _format(fmt)
        return cls._like(torch.empty(0, dtype=torch.uint8, device=device), shape, fmt)

    @classmethod
    def _like(cls, t, shape, fmt: str) -> "MxTensor":
        """An uninitialised one on t's device."""
        x = cls.__new__(cls)
        *lead, x.cols = shape
        x.fmt = fmt
        data, scales = _pitches(x.cols, fmt)
        x.data = t.new_empty((*lead, data), dtype=torch.uint8)
        x.scales = x.data.new_empty((*lead, scales))
        return x

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
    code, format_code = _dtype(values, "values"), _format(fmt)
    if values.dim() == 2:
        rows, cols = values.shape
        stride = _row_stride(values, "values")
    else:
        _need(values.dim() > 2 and values.is_contiguous(), "values must be a matrix, or contiguous with more dimensions")
        cols = stride = values.shape[-1]
        rows = values.numel() // cols if cols else 0
    if out is None:
        index = _index(values)
        out = MxTensor._like(values, values.shape, fmt)
    else:
        _need(out.shape == tuple(values.shape) and out.fmt == fmt, "out has another shape or format")
        index = _index(values, out.data, out.scales)
    _call(load().lm_mx_quantize, index, values.data_ptr(), code, rows, cols, stride, format_code, out.data.data_ptr(), out.scales.data_ptr())
    return out


def mx_dequantize(x: MxTensor, dtype=torch.float32, out=None):
    """lm_mx_dequantize: the values that x stands for, as `dtype`."""
    index = _index(x.data, x.scales, out)
    if out is None:
        out = x.data.new_empty(x.shape, dtype=dtype)
    else:
        _full(out, x.shape, dtype, "out has another shape or type, or is not contiguous")
    _call(load().lm_mx_dequantize, index, x.data.data_ptr(), x.scales.data_ptr(), _FORMATS[x.fmt], x.rows, x.cols, out.data_ptr(), _dtype(out, "out"), x.cols)
    return out


def mx_matmul(x: MxTensor, w: MxTensor, offsets=None, dtype=torch.bfloat16, out=None):
    """lm_mx_matmul: x [rows, k], sorted by group, times the transposed 4-bit w [groups, n, k] of
    each row's group -> [rows, n] of `dtype`.

    offsets: int32 [groups + 1] on the device (SortPlan.offsets); None with one group (w may be
    [n, k] then).  Rows of no group keep what `out` held."""
    wd = w.data.shape
    _need(x.data.dim() == 2 and len(wd) in (2, 3) and w.fmt == "e2m1" and x.cols == w.cols, "x must be [rows, k] and w 4-bit [groups, n, k] with the same k")
    groups = wd[0] if len(wd) == 3 else 1
    rows, n = x.data.shape[0], wd[-2]
    index = _index(x.data, x.scales, w.data, w.scales, offsets, out)
    if offsets is None:
        _need(groups == 1, "several groups need offsets")
    else:
        _need(offsets.dtype == torch.int32 and offsets.is_contiguous() and offsets.numel() == groups + 1, "offsets must be int32 [groups + 1]")
    if out is None:
        out = x.data.new_empty((rows, n), dtype=dtype)
        stride = n
    else:
        _need(tuple(out.shape) == (rows, n) and out.dtype == dtype, "out has another shape or type")
        stride = _row_stride(out, "out")
    _call(load().lm_mx_matmul, index, x.data.data_ptr(), x.scales.data_ptr(), _FORMATS[x.fmt], rows, w.data.data_ptr(), w.scales.data_ptr(), groups, n, x.cols,
          None if offsets is None else offsets.data_ptr(), out.data_ptr(), _dtype(out, "out"), stride)
    return out


def sync(device=None) -> None:
    """lm_ops_sync: waits for the device's current stream and raises if a kernel gave up waiting
    (device: the current one by default, and for "cuda" without an index)."""
    device = torch.device("cuda" if device is None else device)
    _need(device.type == "cuda", "sync needs a CUDA device")
    _call(load().lm_ops_sync, torch.cuda.current_device() if device.index is None else device.index)


def add_rms_norm(hidden, delta, weight, eps: float, fmt: str = "e4m3", bf16: bool = False, out=None):
    """lm_gemm_add_rms_norm_mx: (hidden + delta, its RMS norm as an MxTensor, the norm in bfloat16
    or None).  hidden and delta (may be None): contiguous float32 or bfloat16 [rows, cols]; weight
    float32 [cols].  The sum has hidden's type and goes to `out`, which may be hidden itself."""
    _need(hidden.dim() == 2 and hidden.is_contiguous() and hidden.dtype in _RESIDUAL, "hidden must be contiguous float32 or bfloat16 [rows, cols]")
    _need(delta is None or (delta.shape == hidden.shape and delta.is_contiguous() and delta.dtype in _RESIDUAL),
          "delta must be contiguous float32 or bfloat16 of hidden's shape")
    rows, cols = hidden.shape
    _full(weight, (cols,), torch.float32, "weight must be contiguous float32 [cols]")
    format_code = _format(fmt)
    index = _index(hidden, delta, weight, out)
    if out is None:
        out = torch.empty_like(hidden)
    else:
        _full(out, hidden.shape, hidden.dtype, "out must be contiguous, of hidden's shape and type")
    q = MxTensor._like(hidden, (rows, cols), fmt)
    plain = hidden.new_empty((rows, cols), dtype=torch.bfloat16) if bf16 else None
    _call(load().lm_gemm_add_rms_norm_mx, index, hidden.data_ptr(), _DTYPES[hidden.dtype], None if delta is None else delta.data_ptr(),
          _DTYPES[hidden.dtype if delta is None else delta.dtype], weight.data_ptr(), rows, cols, eps, out.data_ptr(),
          None if plain is None else plain.data_ptr(), format_code, q.data.data_ptr(), q.scales.data_ptr())
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
    index = _index(topk_idx)
    plan = SortPlan.__new__(SortPlan)
    plan.offsets, plan.at = topk_idx.new_empty((experts + 1,)), torch.empty_like(topk_idx)
    tokens, k = topk_idx.shape
    _call(load().lm_moe_sort_plan, index, topk_idx.data_ptr(), tokens, k, experts, plan.offsets.data_ptr(), plan.at.data_ptr())
    return plan


def _sort(x, plan: SortPlan, out):
    x_stride = _row_stride(x, "x")
    (tokens, k), cols = plan.at.shape, x.shape[1]
    _need(x.shape[0] == tokens, "x must have a row for each token of the plan")
    if out is None:
        index = _index(x, plan.at)
        out = x.new_empty((tokens * k, cols))
        out_stride = cols
    else:
        out_stride = _row_stride(out, "out")
        _need(out.dtype == x.dtype and out.shape[1] == cols, "out must have x's type and columns")
        index = _index(x, plan.at, out)
    z = x.element_size()
    _call(load().lm_moe_sort_rows, index, x.data_ptr(), x_stride * z, plan.at.data_ptr(), tokens, k, cols * z, out.data_ptr(), out_stride * z, out.shape[0])
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
    (tokens, k), (n_rows, cols) = plan.at.shape, rows.shape
    if weights is not None:
        _full(weights, (tokens, k), torch.float32, "weights must be contiguous float32 [tokens, top_k]")
    if out is None:
        _need(not accumulate, "accumulate needs out")
        _need(dtype is None or dtype in (rows.dtype, torch.float32), "the result has rows' type or float32")
        index = _index(rows, plan.at, weights)
        out = rows.new_empty((tokens, cols), dtype=dtype)
    else:
        _need(out.dtype in (rows.dtype, torch.float32), "the result has rows' type or float32")
        _full(out, (tokens, cols), dtype or out.dtype, "out must be contiguous [tokens, cols] of the given type")
        index = _index(rows, plan.at, weights, out)
    _call(load().lm_moe_unsort_rows, index, rows.data_ptr(), code, n_rows, plan.at.data_ptr(), None if weights is None else weights.data_ptr(), tokens, k, cols,
          out.data_ptr(), _DTYPES[out.dtype], int(accumulate))
    return out


def sort_rows_backward(grad_rows, plan: SortPlan, out=None, dtype=None):
    """The gradient of sort_rows: grad_x[t] = sum_j grad_rows[at[t, j]]."""
    return unsort_rows(grad_rows, plan, None, out, dtype)


def unsort_rows_backward(grad_y, rows, plan: SortPlan, weights, out=None):
    """lm_moe_unsort_rows_backward: (grad_rows, grad_weights) of unsort_rows with weights.  grad_y has
    rows' type or is float32 (lm_moe_unsort_rows_backward_f32), as the result it belongs to.
    grad_rows goes to `out` (which may be rows itself); rows of no pair keep what it held
    (uninitialised without it)."""
    _need(rows.dim() == 2 and rows.is_contiguous(), "rows must be a contiguous matrix")
    code = _dtype(rows, "rows")
    (tokens, k), (n_rows, cols) = plan.at.shape, rows.shape
    wide = grad_y.dtype == torch.float32 and rows.dtype != torch.float32
    _full(grad_y, (tokens, cols), torch.float32 if wide else rows.dtype, "grad_y must be contiguous [tokens, cols] of rows' type or float32")
    _full(weights, (tokens, k), torch.float32, "weights must be contiguous float32 [tokens, top_k]")
    index = _index(grad_y, rows, plan.at, weights, out)
    if out is None:
        out = torch.empty_like(rows)
    else:
        _full(out, rows.shape, rows.dtype, "out must be contiguous, of rows' shape and type")
    grad_weights = torch.empty_like(weights)
    _call(load().lm_moe_unsort_rows_backward_f32 if wide else load().lm_moe_unsort_rows_backward, index, grad_y.data_ptr(), rows.data_ptr(), code, n_rows, plan.at.data_ptr(), weights.data_ptr(), tokens, k, cols,
          out.data_ptr(), grad_weights.data_ptr())
    return out, grad_weights
