"""The experts' matrix products outside the fused layer (include/megamoe_products.h).

``submission.MoELayer`` runs routing, experts and combine in one launch, with E4M3 or MXFP4
experts. These are the products by themselves, for programs that bring the rows into expert
order on their own: to train or adapt experts in bf16 or fp16 (``grouped_mm``, differentiable),
and to serve experts held in int8 with one scale for each token and each output channel
(``quantize_rows_int8``, ``grouped_int8_mm``, and ``int8_mm`` for a single matrix such as a
shared expert's).

``counts`` (int64 [E], on the GPU) holds the rows of each expert, in order: expert e's rows
start where expert e-1's end. It is read on the device only, so no call waits for the host.
Rows behind the last expert's belong to none: their results are zero, or stay as they were in
``out``. Counts that are negative or add up to more than the rows make the whole result NaN.

Every call is issued on torch's current stream of the inputs' device, as one kernel without a
workspace, and can be captured in a graph after the same call ran once outside. There is no
fallback; bad arguments raise ValueError, tensors off the GPU RuntimeError, a failed launch or
a geometry beyond the limits MegaMoEError.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .submission import _stream_handle

_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}
_HALVES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
_byref, _Product, _Tensor = ctypes.byref, _lib.Product, torch.Tensor


def _device(t, name: str) -> torch.device:
    if not isinstance(t, _Tensor):
        raise ValueError(f"{name}: expected a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"the products run on a GPU; {name} is on {t.device}")
    return t.device


def _dense(t, name: str, dtype, shape, index: int) -> None:
    """``t`` is a contiguous tensor of this type and shape on GPU ``index``, or ValueError."""
    if not isinstance(t, _Tensor):
        raise ValueError(f"{name}: expected a tensor")
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name}: expected {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    if t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous on cuda:{index}")


def _stride(t: torch.Tensor) -> int | None:
    """The row stride of 2-D ``t``, or None if its rows are not dense or overlap."""
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        return None
    if rows <= 1:
        return cols or 1
    return ld if ld >= cols else None


def _rows(t, name: str, dtype, cols, index: int) -> tuple[torch.Tensor, int]:
    """2-D input rows and their stride; rows that are not dense (a broadcast or transposed
    tensor) are copied."""
    if not isinstance(t, _Tensor):
        raise ValueError(f"{name}: expected a tensor")
    if t.dim() != 2 or t.dtype != dtype or (cols is not None and t.shape[1] != cols):
        raise ValueError(f"{name}: expected [rows, {'columns' if cols is None else cols}] {dtype}, "
                         f"got {tuple(t.shape)} {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, expected cuda:{index}")
    ld = _stride(t)
    if ld is None:
        t = t.contiguous()
        ld = max(t.shape[1], 1)
    return t, ld


def _extent(t: torch.Tensor) -> tuple[int, int]:
    """The bytes [first, last) that ``t`` spans."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _given(out, shape, dtype, index: int, inputs) -> int:
    """The row stride of a given result, which may not overlap an input."""
    if not isinstance(out, _Tensor):
        raise ValueError("out: expected a tensor")
    if out.dtype != dtype or out.shape != shape or out.get_device() != index:
        raise ValueError(f"out: expected {tuple(shape)} {dtype} on cuda:{index}, got {tuple(out.shape)} {out.dtype} on "
                         f"{out.device}")
    ld = _stride(out) if out.dim() == 2 else (max(shape[-1], 1) if out.is_contiguous() else None)
    if ld is None:
        raise ValueError("out: its rows must be dense and apart")
    if torch.is_grad_enabled() and out.requires_grad:
        raise ValueError("out: must not require a gradient")
    a, b = _extent(out)
    for t in inputs:
        c, d = _extent(t)
        if a < d and c < b:
            raise ValueError("out: overlaps an input")
    return ld


def _run(name: str, device: torch.device, *args) -> None:
    """One call of the library on torch's current stream of ``device``."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == device.index:
        status = fn(*args, _stream_handle(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _stream_handle(device))
    if status:
        _lib.check(status, name.removeprefix("megamoe_"))


def _grouped(x, weight, counts, transposed: bool, out) -> torch.Tensor:
    device = _device(x, "x")
    index, dtype = device.index, x.dtype
    if dtype not in _HALVES:
        raise ValueError(f"x: expected bfloat16 or float16, got {dtype}")
    if not isinstance(weight, _Tensor) or weight.dim() != 3:
        raise ValueError("weight: expected [experts, out, in] (or [experts, in, out] when transposed)")
    shape = weight.shape
    E, N, K = shape
    if transposed:
        N, K = K, N
    _dense(weight, "weight", dtype, shape, index)
    x, ldx = _rows(x, "x", dtype, K, index)
    _dense(counts, "counts", torch.int64, (E,), index)
    R = x.shape[0]
    if out is None:
        y, ldy = x.new_empty((R, N)), N or 1
    else:
        y, ldy = out, _given(out, (R, N), dtype, index, (x, weight, counts))
    p = _Product(R, E, N, K, _HALVES[dtype], transposed, out is None, ldx, ldy)
    _run("megamoe_grouped_mm", device, _byref(p), x.data_ptr(), weight.data_ptr(), counts.data_ptr(), y.data_ptr())
    return y


def _wgrad(dy, x, counts, out) -> torch.Tensor:
    device = _device(x, "x")
    index, dtype = device.index, x.dtype
    if dtype not in _HALVES:
        raise ValueError(f"x: expected bfloat16 or float16, got {dtype}")
    x, ldx = _rows(x, "x", dtype, None, index)
    dy, ldy = _rows(dy, "dy", dtype, None, index)
    R, K = x.shape
    if dy.shape[0] != R:
        raise ValueError(f"dy: {dy.shape[0]} rows, x has {R}")
    if not isinstance(counts, _Tensor) or counts.dim() != 1:
        raise ValueError("counts: expected int64 [experts]")
    E, N = counts.shape[0], dy.shape[1]
    _dense(counts, "counts", torch.int64, (E,), index)
    if out is None:
        dw = x.new_empty((E, N, K))
    else:
        dw = out
        _given(out, (E, N, K), dtype, index, (x, dy, counts))
    p = _Product(R, E, N, K, _HALVES[dtype], 0, 0, ldx, ldy)
    _run("megamoe_grouped_mm_wgrad", device, _byref(p), dy.data_ptr(), x.data_ptr(), counts.data_ptr(), dw.data_ptr())
    return dw


# The product and the weight's gradient are bilinear and each other's derivatives: the gradients
# of either are again one of the two, so both can be differentiated any number of times.

class _GroupedMM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, counts, transposed):
        ctx.save_for_backward(x, weight, counts)
        ctx.transposed = transposed
        return _grouped(x, weight, counts, transposed, None)

    @staticmethod
    def backward(ctx, dy):
        x, weight, counts = ctx.saved_tensors
        wants_x, wants_w, _, _ = ctx.needs_input_grad
        dx = grouped_mm(dy, weight, counts, transposed=not ctx.transposed) if wants_x else None
        dw = None
        if wants_w:
            dw = grouped_mm_wgrad(x, dy, counts) if ctx.transposed else grouped_mm_wgrad(dy, x, counts)
        return dx, dw, None, None


class _WGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dy, x, counts):
        ctx.save_for_backward(dy, x, counts)
        return _wgrad(dy, x, counts, None)

    @staticmethod
    def backward(ctx, g):
        dy, x, counts = ctx.saved_tensors
        g = g.contiguous()
        wants_dy, wants_x, _ = ctx.needs_input_grad
        return (grouped_mm(x, g, counts) if wants_dy else None,
                grouped_mm(dy, g, counts, transposed=True) if wants_x else None, None)


def _differentiable(out, *tensors) -> bool:
    """Whether a call on ``tensors`` is to be recorded; it cannot write to a given tensor then."""
    if not torch.is_grad_enabled() or not any(isinstance(t, _Tensor) and t.requires_grad for t in tensors):
        return False
    if out is not None:
        raise ValueError("out: the result of inputs that require gradients cannot be written to a given tensor")
    return True


def grouped_mm(x: torch.Tensor, weight: torch.Tensor, counts: torch.Tensor, *, transposed: bool = False,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """y [R, N]: row r of expert e is ``weight[e] @ x[r]`` (weight [E, N, K]) or, ``transposed``,
    ``x[r] @ weight[e]`` (weight [E, K, N]); bf16 or fp16, summed in fp32, rounded once.

    ``x`` [R, K] may have any row stride (rows that are not dense are copied); ``weight`` is
    dense. Differentiable in ``x`` and ``weight`` unless ``out`` is given, which takes the result
    and keeps its rows of no expert."""
    if _differentiable(out, x, weight):
        return _GroupedMM.apply(x, weight, counts, bool(transposed))
    return _grouped(x, weight, counts, bool(transposed), out)


def grouped_mm_wgrad(dy: torch.Tensor, x: torch.Tensor, counts: torch.Tensor, *,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """dw [E, N, K]: the gradient of ``grouped_mm``'s weight, ``dy[r]^T x[r]`` summed over each
    expert's rows (dy [R, N], x [R, K]; exchange them for a transposed weight), bf16 or fp16, summed
    in fp32. Experts without rows get zero. Differentiable in ``dy`` and ``x`` unless ``out`` is
    given."""
    if _differentiable(out, dy, x):
        return _WGrad.apply(dy, x, counts)
    return _wgrad(dy, x, counts, out)


def _int8(x, x_scale, weight, weight_scale, counts, out_dtype, out) -> torch.Tensor:
    device = _device(x, "x")
    index = device.index
    kind = _TYPES.get(out_dtype)
    if kind is None:
        raise ValueError(f"out_dtype: expected bfloat16, float16 or float32, got {out_dtype}")
    shape = weight.shape
    N, K = shape[-2:]
    x, ldx = _rows(x, "x", torch.int8, K, index)
    R = x.shape[0]
    _dense(x_scale, "x_scale", torch.float32, (R,), index)
    _dense(weight, "weight", torch.int8, shape, index)
    _dense(weight_scale, "weight_scale", torch.float32, shape[:-1], index)
    if counts is None:
        E, counts_at = 1, None
    else:
        E = shape[0]
        _dense(counts, "counts", torch.int64, (E,), index)
        counts_at = counts.data_ptr()
    if out is None:
        y, ldy = torch.empty((R, N), dtype=out_dtype, device=device), N or 1
    else:
        inputs = (x, x_scale, weight, weight_scale) + (() if counts is None else (counts,))
        y, ldy = out, _given(out, (R, N), out_dtype, index, inputs)
    p = _Product(R, E, N, K, kind, 0, out is None, ldx, ldy)
    _run("megamoe_int8_mm", device, _byref(p), x.data_ptr(), x_scale.data_ptr(), weight.data_ptr(),
         weight_scale.data_ptr(), counts_at, y.data_ptr())
    return y


def int8_mm(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
            out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """y [R, N] = (x @ weight^T) * x_scale[:, None] * weight_scale[None, :]: x int8 [R, K] with
    fp32 scales [R], weight int8 [N, K] (out features by in features) with fp32 scales [N]. The
    integer sums are exact; the result is bf16, fp16 or fp32."""
    _device(x, "x")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight: expected int8 [out, in]")
    return _int8(x, x_scale, weight, weight_scale, None, out_dtype, out)


def grouped_int8_mm(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                    counts: torch.Tensor, *, out_dtype: torch.dtype = torch.bfloat16,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """``int8_mm`` of every expert's rows with its own matrix: weight int8 [E, N, K] with fp32
    scales [E, N], rows grouped by ``counts`` as in ``grouped_mm``."""
    _device(x, "x")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 3:
        raise ValueError("weight: expected int8 [experts, out, in]")
    if not isinstance(counts, torch.Tensor):
        raise ValueError("counts: expected int64 [experts]")
    return _int8(x, x_scale, weight, weight_scale, counts, out_dtype, out)


def quantize_rows_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """int8 payload [R, C] and fp32 scales [R] of bf16, fp16 or fp32 rows: with a the row's
    largest magnitude (at least 2^-100), scale = a / 127 and q = x * (127 / a) rounded to nearest
    even. A row with NaN or an infinity gets the scale NaN and zeros."""
    device = _device(x, "x")
    kind = _TYPES.get(x.dtype)
    if kind is None or x.dim() != 2:
        raise ValueError("quantize_rows_int8 takes 2-D bfloat16, float16 or float32 rows")
    x, ld = _rows(x, "x", x.dtype, None, device.index)
    rows, cols = shape = x.shape
    q = torch.empty(shape, dtype=torch.int8, device=device)
    scale = torch.empty((rows,), dtype=torch.float32, device=device)
    _run("megamoe_quantize_rows_int8", device, rows, cols, ld, kind, x.data_ptr(), q.data_ptr(), scale.data_ptr())
    return q, scale
