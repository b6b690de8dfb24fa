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
be captured).  Forward-mode tangents are refused everywhere.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


class TokenOrder:
    """Where a batch's (token, slot) units went: ``starts [E+1]`` (first row of
    each expert; ``starts[E]`` rows are in use), ``row_of [T, k]`` (row of each
    unit, -1 for none), ``unit_of [T*k]`` (unit ``t*k + j`` of each row, -1 past
    the last).  int32 CUDA tensors."""

    __slots__ = ("_buf", "_starts", "_row_of", "_unit_of", "shape", "num_experts", "device")

    def __init__(self, starts, row_of, unit_of):
        for name, t, dim in (("starts", starts, 1), ("row_of", row_of, 2), ("unit_of", unit_of, 1)):
            if t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dim}-d int32 tensor")
            if t.device != starts.device:
                raise ValueError("starts, row_of and unit_of must be on one device")
        if starts.numel() < 2 or unit_of.numel() != row_of.numel():
            raise ValueError("starts needs E + 1 entries and unit_of one per unit of row_of")
        self._buf = None
        self._starts, self._row_of, self._unit_of = starts, row_of, unit_of
        self.shape, self.num_experts, self.device = tuple(row_of.shape), starts.numel() - 1, starts.device

    @classmethod
    def _new(cls, t, k, num_experts, like):
        """An order to be filled in: one buffer, row_of then unit_of then starts."""
        self = cls.__new__(cls)
        self._buf = like.new_empty(2 * t * k + num_experts + 1, dtype=torch.int32)
        self._starts = self._row_of = self._unit_of = None
        self.shape, self.num_experts, self.device = (t, k), num_experts, like.device
        return self

    def _pointers(self):
        """Addresses of (row_of, unit_of, starts)."""
        if self._buf is None:
            return self._row_of.data_ptr(), self._unit_of.data_ptr(), self._starts.data_ptr()
        p, u = self._buf.data_ptr(), 4 * self.shape[0] * self.shape[1]
        return p, p + u, p + 2 * u

    @property
    def row_of(self):
        if self._row_of is None:
            t, k = self.shape
            self._row_of = self._buf.as_strided((t, k), (k, 1), 0)
        return self._row_of

    @property
    def unit_of(self):
        if self._unit_of is None:
            n = self.shape[0] * self.shape[1]
            self._unit_of = self._buf.as_strided((n,), (1,), n)
        return self._unit_of

    @property
    def starts(self):
        if self._starts is None:
            self._starts = self._buf.as_strided((self.num_experts + 1,), (1,), 2 * self.shape[0] * self.shape[1])
        return self._starts

    def get_device(self):
        return self.device.index if self.device.type == "cuda" else -1

    def record_stream(self, stream):
        for t in (self._buf, self._starts, self._row_of, self._unit_of):
            if t is not None:
                t.record_stream(stream)


try:  # the handle alone, without a Stream object (3 us of a call's 15 on the host)
    _stream_handle = torch._C._cuda_getCurrentRawStream
    _current_device = torch._C._cuda_getDevice  # (there is a CUDA tensor: nothing to initialise)
except AttributeError:
    _current_device = torch.cuda.current_device

    def _stream_handle(device):
        return torch.cuda.current_stream(device).cuda_stream


def _on(stream, fn, tensors, args):
    """``fn(*args, stream handle)`` with the tensors' device current and ``stream``
    (default: that device's current stream) as its current stream, so that
    outputs and scratch belong to the stream that uses them."""
    at = tensors[0].get_device()  # the index alone, without a device object
    if at < 0:
        raise ValueError(f"tensors must be on a CUDA device, got {tensors[0].device}")
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError(f"tensors are on {tensors[0].device} and {t.device}")
    if stream is None and _current_device() == at:
        return fn(*args, _stream_handle(at))
    dev = tensors[0].device
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


def _output(out, shape, dtype, like, name="out"):
    if dtype not in _DT:
        raise ValueError(f"{name}: unsupported dtype {dtype} (float32 or bfloat16)")
    if out is None:
        return like.new_empty(shape, dtype=dtype), shape[1]
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"{name} must be {tuple(shape)} {dtype}, got {tuple(out.shape)} {out.dtype}")
    if out.device != like.device:
        raise ValueError(f"{name} is on {out.device}, expected {like.device}")
    if shape[1] > 1 and out.stride(1) != 1 or shape[0] > 1 and out.stride(0) < shape[1]:
        raise ValueError(f"{name} needs rows of unit stride that do not overlap")
    return out, out.stride(0) if shape[0] > 1 else shape[1]


def _overlap(a, b):
    """Whether two matrices of unit column stride may share bytes (column ranges
    of one row-strided buffer do not)."""
    ea, eb = a.element_size(), b.element_size()
    la, lb = a.stride(0) * ea, b.stride(0) * eb
    a0, b0 = a.data_ptr(), b.data_ptr()
    if not a.numel() or not b.numel():
        return False
    if b0 >= a0 + (a.shape[0] - 1) * la + a.shape[1] * ea or a0 >= b0 + (b.shape[0] - 1) * lb + b.shape[1] * eb:
        return False
    if la != lb or la == 0:
        return True
    at = (b0 - a0) % la
    return not (at >= a.shape[1] * ea and at + b.shape[1] * eb <= la)


def _apart(out, *tensors):
    """Refuses an output given by the caller that overlaps an input."""
    if out is not None and any(t is not None and _overlap(out, t) for t in tensors):
        raise ValueError("out overlaps an input")


def _ids(ids, num_experts):
    if ids.dtype != torch.int32 or ids.dim() != 2:
        raise ValueError(f"expert ids must be [T, k] int32, got {tuple(ids.shape)} {ids.dtype}")
    if not 1 <= num_experts <= _lib.MAX_EXPERTS:
        raise ValueError(f"num_experts={num_experts} outside [1, {_lib.MAX_EXPERTS}]")
    if not 1 <= ids.shape[1] <= _lib.MAX_TOPK:
        raise ValueError(f"k={ids.shape[1]} outside [1, {_lib.MAX_TOPK}]")


def _weights(weights, shape, name="weights"):
    if weights.dtype != torch.float32 or tuple(weights.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)} float32, got {tuple(weights.shape)} {weights.dtype}")
    if shape[1] > 1 and weights.stride(1) != 1:
        weights = weights.contiguous()
    return weights, weights.stride(0) if shape[0] > 1 else shape[1]


def _capturing(stream):
    if stream is None:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def _apply(fn, stream, *args):
    """``fn.apply`` on ``stream``: autograd runs the backward pass on the stream that
    was current here, which so is the one that owns what the forward pass kept."""
    if stream is None:
        return fn.apply(*args, None)
    with torch.cuda.stream(stream):
        return fn.apply(*args, stream)


def _no_tangent(what, *tensors):
    """Refuses dual tensors: no call carries forward-mode tangents."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode gradient")


def _differentiable(what, out, stream, *tensors):
    _no_tangent(what, *tensors)
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors):
        return False
    if out is not None:
        raise RuntimeError(f"{what}: out= does not take part in autograd, but an input requires a gradient")
    if _capturing(stream):
        raise RuntimeError(f"{what}: the differentiable form cannot be captured into a CUDA graph; "
                           "capture detached tensors and the *_backward call")
    return True


# ------------------------------------------------------------------ the calls
def _sort_and_move(x, ldx, ids, num_experts, rows, ldr, s):
    L = _lib.lib()
    t, k = ids.shape
    order = TokenOrder._new(t, k, num_experts, ids)
    row_of, unit_of, starts = order._pointers()
    ws, need = None, 0
    if t * k > 1024:  # smaller batches need no scratch
        need = L.aem_token_sort_workspace(t, k, num_experts)
        keep = ids.new_empty(need // 4)
        ws = keep.data_ptr()
    st, sk = ids.stride()
    if x is None:
        _lib.check(L.aem_token_sort(ids.data_ptr(), t, k, st, sk, num_experts, starts, row_of, unit_of, ws,
                                    need, s), "aem_token_sort")
    else:
        _lib.check(L.aem_dispatch(x.data_ptr(), _DT[x.dtype], ldx, x.shape[1], ids.data_ptr(), t, k, st, sk,
                                  num_experts, rows.data_ptr(), ldr, starts, row_of, unit_of, ws, need, s),
                   "aem_dispatch")
    return order


def _dispatch(x, ids, num_experts, out, s):
    x, ldx = _matrix(x, "x", rows=ids.shape[0])
    if x.shape[1] == 0:
        raise ValueError("x has no columns")
    rows, ldr = _output(out, (ids.numel(), x.shape[1]), x.dtype, x, "rows")
    _apart(out, x)
    return rows, _sort_and_move(x, ldx, ids, num_experts, rows, ldr, s)


def _dispatch_rows(x, order, out, s):
    t, k = order.shape
    x, ldx = _matrix(x, "x", rows=t)
    rows, ldr = _output(out, (t * k, x.shape[1]), x.dtype, x, "rows")
    _apart(out, x)
    row_of, _, starts = order._pointers()
    _lib.check(_lib.lib().aem_dispatch_rows(x.data_ptr(), _DT[x.dtype], ldx, x.shape[1], row_of, starts, t, k,
                                            order.num_experts, rows.data_ptr(), ldr, s),
               "aem_dispatch_rows")
    return rows


def _combine(rows, weights, order, out_dtype, out, s):
    t, k = order.shape
    rows, ldr = _matrix(rows, "rows", rows=t * k)
    d = rows.shape[1]
    ldw = 0
    if weights is not None:
        weights, ldw = _weights(weights, (t, k))
    given = out
    out, ldo = _output(out, (t, d), out_dtype or (rows.dtype if out is None else out.dtype), rows)
    _apart(given, rows, weights)
    _lib.check(_lib.lib().aem_combine(rows.data_ptr(), _DT[rows.dtype], ldr,
                                      None if weights is None else weights.data_ptr(), ldw,
                                      order._pointers()[0], t, k, d, out.data_ptr(),
                                      _DT[out.dtype], ldo, s), "aem_combine")
    return out


def _combine_backward(grad_out, rows, weights, order, rows_dtype, want_rows, want_weights, s):
    t, k = order.shape
    row_of, _, starts = order._pointers()
    grad_out, ldg = _matrix(grad_out, "grad_out", rows=t)
    d = grad_out.shape[1]
    ldr = ldw = ldgr = 0
    grad_rows = grad_weights = None
    if want_weights:
        rows, ldr = _matrix(rows, "rows", d=d, rows=t * k)
        rows_dtype = rows.dtype
        grad_weights = grad_out.new_empty((t, k), dtype=torch.float32)
    if weights is not None:
        weights, ldw = _weights(weights, (t, k))
    if want_rows:
        grad_rows, ldgr = _output(None, (t * k, d), rows_dtype, grad_out, "grad_rows")
    _lib.check(_lib.lib().aem_combine_backward(
        grad_out.data_ptr(), _DT[grad_out.dtype], ldg, rows.data_ptr() if want_weights else None,
        _DT[rows_dtype], ldr, None if weights is None else weights.data_ptr(), ldw, row_of, starts, t, k, order.num_experts, d,
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
            rows = _on(stream, _dispatch_rows, (x, order), (x, order, None))
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
        out = _on(stream, _combine, (rows, weights, order), (rows, weights, order, out_dtype, None))
        ctx.save_for_backward(rows, weights)
        ctx.order = order
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _refuse_capture("combine")
        rows, weights = ctx.saved_tensors
        gr, gw = _on(None, _combine_backward, (grad, rows, weights, ctx.order),
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
    if _differentiable("dispatch", out, stream, x):
        holder = []
        rows = _apply(_DispatchFn, stream, x, ids, num_experts, None, holder)
        return rows, holder[0]
    return _on(stream, _dispatch, (x, ids, out), (x, ids, num_experts, out))


def dispatch_rows(x, order, out=None, stream=None):
    """Rows of another ``x [T, d]`` by an existing order."""
    if _differentiable("dispatch_rows", out, stream, x):
        return _apply(_DispatchFn, stream, x, None, 0, order, None)
    return _on(stream, _dispatch_rows, (x, order, out), (x, order, out))


def dispatch_backward(grad_rows, order, out_dtype=None, out=None, stream=None):
    """Gradient of ``dispatch``: ``grad_x[t] = sum_j grad_rows[row_of[t, j]]``."""
    _no_tangent("dispatch_backward", grad_rows)
    return _on(stream, _combine, (grad_rows, order, out), (grad_rows, None, order, out_dtype, out))


def combine(rows, weights, order, out_dtype=None, out=None, stream=None):
    """``out[t] = sum_j weights[t, j] * rows[row_of[t, j]]`` (``rows [T*k, d]``,
    ``weights [T, k]`` float32 or ``None`` for 1; ``out_dtype`` defaults to the
    rows')."""
    if _differentiable("combine", out, stream, rows, weights):
        return _apply(_CombineFn, stream, rows, weights, order, out_dtype)
    return _on(stream, _combine, (rows, weights, order, out), (rows, weights, order, out_dtype, out))


def combine_backward(grad_out, rows, weights, order, stream=None):
    """Gradients of ``combine``: ``(grad_rows [T*k, d]`` in the rows' dtype,
    ``grad_weights [T, k]`` float32``)``."""
    _no_tangent("combine_backward", grad_out, rows, weights)
    return _on(stream, _combine_backward, (grad_out, rows, weights, order),
               (grad_out, rows, weights, order, rows.dtype, True, True))
