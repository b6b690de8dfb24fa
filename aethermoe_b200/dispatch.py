"""Token dispatch and combine around expert products, with their gradients.

For callers that run their own experts between the framework's gating and
its combine: ``dispatch`` sorts the tokens by expert and copies their rows,
``combine`` weights the experts' rows and sums them per token.

    idx, val = gating(...)                                   # [T, k] int32, [T, k] float32
    rows, order = dispatch(x, idx, num_experts)              # [T*k, d], TokenOrder
    y = experts(rows, order.starts)                          # e.g. q4.grouped_q4_matmul
    out = combine(y, val, order)                             # [T, d]

Tensors are torch CUDA tensors; every kernel is in ``libaethermoe.so``
(``aem_dispatch`` and the following calls of ``include/aem.h``, which define
the results).  A negative expert id is a unit without an expert: no row, no
contribution, zero gradients.  ``dispatch``, ``dispatch_rows`` and ``combine``
take part in autograd when an input requires a gradient; a training step that
is captured into a CUDA graph calls ``dispatch_backward`` and
``combine_backward`` itself, because autograd's accumulation into leaves runs
on streams that the capture does not own (the differentiable forms refuse to
be captured).
"""
from __future__ import annotations

import torch

from . import _lib

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


class TokenOrder:
    """Where a batch's (token, slot) units went: ``starts [E+1]`` (first row of
    each expert; ``starts[E]`` rows are in use), ``row_of [T, k]`` (row of each
    unit, -1 for none), ``unit_of [T*k]`` (unit ``t*k + j`` of each row, -1 past
    the last).  int32 CUDA tensors."""

    __slots__ = ("starts", "row_of", "unit_of")

    def __init__(self, starts, row_of, unit_of):
        for name, t, dim in (("starts", starts, 1), ("row_of", row_of, 2), ("unit_of", unit_of, 1)):
            if t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dim}-d int32 tensor")
            if t.device != starts.device:
                raise ValueError("starts, row_of and unit_of must be on one device")
        if starts.numel() < 2 or unit_of.numel() != row_of.numel():
            raise ValueError("starts needs E + 1 entries and unit_of one per unit of row_of")
        self.starts, self.row_of, self.unit_of = starts, row_of, unit_of

    @property
    def num_experts(self):
        return self.starts.numel() - 1


def _on(stream, fn, tensors, args):
    """``fn(*args, stream handle)`` with the tensors' device current and ``stream``
    (default: that device's current stream) as its current stream, so that
    outputs and scratch belong to the stream that uses them."""
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, got {dev}")
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors are on {dev} and {t.device}")
    if stream is None and torch.cuda.current_device() == dev.index:
        return fn(*args, torch.cuda.current_stream().cuda_stream)
    if stream is None:
        stream = torch.cuda.current_stream(dev)
    elif stream.device != dev:
        raise ValueError(f"stream is on {stream.device}, the tensors on {dev}")
    with torch.cuda.stream(stream):  # switches the device too
        out = fn(*args, stream.cuda_stream)
        for t in tensors:
            if t is not None:
                t.record_stream(stream)
    return out


def _matrix(t, name, d=None, rows=None):
    """``t`` as a row-strided matrix (unit column stride) and its row stride."""
    if t.dtype not in _DT:
        raise ValueError(f"{name}: unsupported dtype {t.dtype} (float32 or bfloat16)")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-d, got shape {tuple(t.shape)}")
    if d is not None and t.shape[1] != d:
        raise ValueError(f"{name} has {t.shape[1]} columns, expected {d}")
    if rows is not None and t.shape[0] != rows:
        raise ValueError(f"{name} has {t.shape[0]} rows, expected {rows}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _output(out, shape, dtype, device, name="out"):
    if out is None:
        if dtype not in _DT:
            raise ValueError(f"{name}: unsupported dtype {dtype} (float32 or bfloat16)")
        return torch.empty(shape, dtype=dtype, device=device), shape[1]
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"{name} must be {tuple(shape)} {dtype}, got {tuple(out.shape)} {out.dtype}")
    if out.device != device:
        raise ValueError(f"{name} is on {out.device}, expected {device}")
    if shape[1] > 1 and out.stride(1) != 1 or shape[0] > 1 and out.stride(0) < shape[1]:
        raise ValueError(f"{name} needs rows of unit stride that do not overlap")
    return out, out.stride(0) if shape[0] > 1 else shape[1]


def _ids(ids, num_experts):
    if ids.dtype != torch.int32 or ids.dim() != 2:
        raise ValueError(f"expert ids must be [T, k] int32, got {tuple(ids.shape)} {ids.dtype}")
    if not 1 <= num_experts <= _lib.MAX_EXPERTS:
        raise ValueError(f"num_experts={num_experts} outside [1, {_lib.MAX_EXPERTS}]")
    if not 1 <= ids.shape[1] <= _lib.MAX_TOPK:
        raise ValueError(f"k={ids.shape[1]} outside [1, {_lib.MAX_TOPK}]")


def _weights(weights, shape):
    if weights.dtype != torch.float32 or tuple(weights.shape) != tuple(shape):
        raise ValueError(f"weights must be {tuple(shape)} float32, got {tuple(weights.shape)} {weights.dtype}")
    if shape[1] > 1 and weights.stride(1) != 1:
        weights = weights.contiguous()
    return weights, weights.stride(0) if shape[0] > 1 else shape[1]


def _differentiable(what, out, *tensors):
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors):
        return False
    if out is not None:
        raise RuntimeError(f"{what}: out= does not take part in autograd, but an input requires a gradient")
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: the differentiable form cannot be captured into a CUDA graph; "
                           "capture detached tensors and the *_backward call")
    return True


# ------------------------------------------------------------------ the calls
def _sort_and_move(x, ldx, ids, num_experts, rows, ldr, s):
    L = _lib.lib()
    t, k = ids.shape
    dev = ids.device
    starts = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    row_of = torch.empty((t, k), dtype=torch.int32, device=dev)
    unit_of = torch.empty(t * k, dtype=torch.int32, device=dev)
    need = L.aem_token_sort_workspace(t, k, num_experts)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    st, sk = ids.stride()
    if x is None:
        _lib.check(L.aem_token_sort(ids.data_ptr(), t, k, st, sk, num_experts, starts.data_ptr(),
                                    row_of.data_ptr(), unit_of.data_ptr(),
                                    ws.data_ptr() if need else None, need, s), "aem_token_sort")
    else:
        _lib.check(L.aem_dispatch(x.data_ptr(), _DT[x.dtype], ldx, x.shape[1], ids.data_ptr(), t, k,
                                  st, sk, num_experts, rows.data_ptr(), ldr, starts.data_ptr(),
                                  row_of.data_ptr(), unit_of.data_ptr(),
                                  ws.data_ptr() if need else None, need, s), "aem_dispatch")
    order = TokenOrder.__new__(TokenOrder)
    order.starts, order.row_of, order.unit_of = starts, row_of, unit_of
    return order


def _dispatch(x, ids, num_experts, out, s):
    x, ldx = _matrix(x, "x", rows=ids.shape[0])
    if x.shape[1] == 0:
        raise ValueError("x has no columns")
    rows, ldr = _output(out, (ids.numel(), x.shape[1]), x.dtype, x.device, "rows")
    return rows, _sort_and_move(x, ldx, ids, num_experts, rows, ldr, s)


def _dispatch_rows(x, order, out, s):
    t, k = order.row_of.shape
    x, ldx = _matrix(x, "x", rows=t)
    rows, ldr = _output(out, (t * k, x.shape[1]), x.dtype, x.device, "rows")
    _lib.check(_lib.lib().aem_dispatch_rows(x.data_ptr(), _DT[x.dtype], ldx, x.shape[1],
                                            order.row_of.data_ptr(), order.starts.data_ptr(), t, k,
                                            order.num_experts, rows.data_ptr(), ldr, s),
               "aem_dispatch_rows")
    return rows


def _combine(rows, weights, order, out_dtype, out, s):
    t, k = order.row_of.shape
    rows, ldr = _matrix(rows, "rows", rows=t * k)
    d = rows.shape[1]
    ldw = 0
    if weights is not None:
        weights, ldw = _weights(weights, (t, k))
    out, ldo = _output(out, (t, d), out_dtype or (rows.dtype if out is None else out.dtype), rows.device)
    _lib.check(_lib.lib().aem_combine(rows.data_ptr(), _DT[rows.dtype], ldr,
                                      None if weights is None else weights.data_ptr(), ldw,
                                      order.row_of.data_ptr(), t, k, d, out.data_ptr(),
                                      _DT[out.dtype], ldo, s), "aem_combine")
    return out


def _combine_backward(grad_out, rows, weights, order, rows_dtype, want_rows, want_weights, s):
    t, k = order.row_of.shape
    grad_out, ldg = _matrix(grad_out, "grad_out", rows=t)
    d = grad_out.shape[1]
    ldr = ldw = ldgr = 0
    grad_rows = grad_weights = None
    if want_weights:
        rows, ldr = _matrix(rows, "rows", d=d, rows=t * k)
        rows_dtype = rows.dtype
        grad_weights = torch.empty((t, k), dtype=torch.float32, device=grad_out.device)
    weights, ldw = _weights(weights, (t, k))
    if want_rows:
        grad_rows, ldgr = _output(None, (t * k, d), rows_dtype, grad_out.device, "grad_rows")
    _lib.check(_lib.lib().aem_combine_backward(
        grad_out.data_ptr(), _DT[grad_out.dtype], ldg, rows.data_ptr() if want_weights else None,
        _DT[rows_dtype], ldr, weights.data_ptr(), ldw, order.row_of.data_ptr(),
        order.starts.data_ptr(), t, k, order.num_experts, d,
        grad_rows.data_ptr() if want_rows else None, ldgr,
        grad_weights.data_ptr() if want_weights else None, s), "aem_combine_backward")
    return grad_rows, grad_weights


class _DispatchFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, num_experts, order, holder, stream):
        if order is None:
            rows, order = _on(stream, _dispatch, (x, ids), (x, ids, num_experts, None))
            holder.append(order)
        else:
            rows = _on(stream, _dispatch_rows, (x, order.row_of), (x, order, None))
        ctx.order, ctx.x_dtype = order, x.dtype
        return rows

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _refuse_capture("dispatch")
        return dispatch_backward(grad, ctx.order, ctx.x_dtype), None, None, None, None, None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order, out_dtype, stream):
        out = _on(stream, _combine, (rows, weights, order.row_of), (rows, weights, order, out_dtype, None))
        ctx.save_for_backward(rows, weights)
        ctx.order = order
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _refuse_capture("combine")
        rows, weights = ctx.saved_tensors
        gr, gw = _on(None, _combine_backward, (grad, rows, weights, ctx.order.row_of),
                     (grad, rows, weights, ctx.order, rows.dtype, ctx.needs_input_grad[0],
                      ctx.needs_input_grad[1]))
        return gr, gw, None, None, None


def _refuse_capture(what):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: its backward cannot be captured into a CUDA graph; "
                           f"call {what}_backward")


def sort_tokens(ids, num_experts, stream=None):
    """The ``TokenOrder`` of expert ids ``[T, k]`` (int32, any strides: a slice of
    gating's ``[T, k+1]`` or a transposed slot-major tensor)."""
    _ids(ids, num_experts)
    return _on(stream, _sort_and_move, (ids,), (None, 0, ids, num_experts, None, 0))


def dispatch(x, ids, num_experts, out=None, stream=None):
    """``(rows [T*k, d], TokenOrder)``: token ``t``'s row of ``x [T, d]`` at every
    ``order.row_of[t, j]``; rows from ``order.starts[E]`` on are zero."""
    _ids(ids, num_experts)
    if _differentiable("dispatch", out, x):
        holder = []
        rows = _DispatchFn.apply(x, ids, num_experts, None, holder, stream)
        return rows, holder[0]
    return _on(stream, _dispatch, (x, ids), (x, ids, num_experts, out))


def dispatch_rows(x, order, out=None, stream=None):
    """Rows of another ``x [T, d]`` by an existing order."""
    if _differentiable("dispatch_rows", out, x):
        return _DispatchFn.apply(x, None, 0, order, None, stream)
    return _on(stream, _dispatch_rows, (x, order.row_of), (x, order, out))


def dispatch_backward(grad_rows, order, out_dtype=None, out=None, stream=None):
    """Gradient of ``dispatch``: ``grad_x[t] = sum_j grad_rows[row_of[t, j]]``."""
    return _on(stream, _combine, (grad_rows, order.row_of), (grad_rows, None, order, out_dtype, out))


def combine(rows, weights, order, out_dtype=None, out=None, stream=None):
    """``out[t] = sum_j weights[t, j] * rows[row_of[t, j]]`` (``rows [T*k, d]``,
    ``weights [T, k]`` float32; ``out_dtype`` defaults to the rows')."""
    if _differentiable("combine", out, rows, weights):
        return _CombineFn.apply(rows, weights, order, out_dtype, stream)
    return _on(stream, _combine, (rows, weights, order.row_of), (rows, weights, order, out_dtype, out))


def combine_backward(grad_out, rows, weights, order, stream=None):
    """Gradients of ``combine``: ``(grad_rows [T*k, d]`` in the rows' dtype,
    ``grad_weights [T, k]`` float32``)``."""
    return _on(stream, _combine_backward, (grad_out, rows, weights, order.row_of),
               (grad_out, rows, weights, order, rows.dtype, True, True))
