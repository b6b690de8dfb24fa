"""8-bit floating point (e4m3) with a scale per block of 128: quantisation of rows
and weights, the packed weight, and the products of rows with it, dense and
grouped by expert, with the gradient of the rows.

    q, s = quantize_fp8_weight(w)                # w [K, N] or [G, K, N], blocks of 128 x 128
    weight = Fp8Weight(q, s)                     # packed once, about K*N bytes a group
    y = fp8_matmul(x, weight)                    # x [M, K], quantised in the call
    rows = quantize_fp8(x)                       # or once for several products
    h = grouped_fp8_matmul(rows, weight, order.starts, out_dtype=torch.bfloat16)

Tensors are torch CUDA tensors; every kernel is in ``libaethermoe.so``
(``aem_quantize_fp8`` and the following calls of ``include/aem.h``, which define
the results).  The products take part in autograd when ``x`` is a tensor that
requires a gradient: the rounding of x passes its gradient on unchanged, and the
gradient is the product of the gradient's own rows, quantised the same way, with
the transposed weight, from the same packed copy.  The weights themselves have no
gradient.  ``fp8_matmul_backward`` and ``grouped_fp8_matmul_backward`` are the
same gradients as plain calls, for a step that is captured into a CUDA graph (the
differentiable forms refuse to be captured).  Forward-mode tangents are refused.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .dispatch import _DT, _apart, _apply, _differentiable, _matrix, _no_tangent, _on, _output, _refuse_capture

BLOCK = 128
_E4M3 = torch.float8_e4m3fn


def _blocks(n):
    return -(-n // BLOCK)


def _no_gradient(what, x, name):
    _no_tangent(what, x)
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no gradient: detach {name} or call it under torch.no_grad()")


class Fp8Rows:
    """Rows in blocks of 128: ``q [M, K]`` float8_e4m3fn and ``scale [M,
    ceil(K/128)]`` float32, CUDA tensors; row m, block b stands for
    ``q[m, 128 b: 128 (b+1)] * scale[m, b]``.  ``quantize_fp8`` makes them; others are
    taken as they are where the products can read them (rows a multiple of 16 bytes
    apart, scales a multiple of 4) and copied otherwise."""

    __slots__ = ("q", "scale", "shape", "device")

    def __init__(self, q, scale):
        if q.dtype != _E4M3 or q.dim() != 2:
            raise ValueError(f"q must be [M, K] float8_e4m3fn, got {tuple(q.shape)} {q.dtype}")
        want = (q.shape[0], _blocks(q.shape[1]))
        if scale.dtype != torch.float32 or tuple(scale.shape) != want:
            raise ValueError(f"scale must be {want} float32, got {tuple(scale.shape)} {scale.dtype}")
        if scale.device != q.device:
            raise ValueError(f"q and scale are on {q.device} and {scale.device}")
        _no_gradient("Fp8Rows", q, "q")
        _no_gradient("Fp8Rows", scale, "scale")
        self._set(q, scale)

    def _set(self, q, scale):
        self.q, self.scale, self.shape, self.device = q, scale, q.shape, q.device
        return self

    def get_device(self):
        return self.q.get_device()

    def record_stream(self, stream):
        self.q.record_stream(stream)
        self.scale.record_stream(stream)


def _new_rows(m, k, like):
    ldq, lds = -(-k // 16) * 16, -(-_blocks(k) // 4) * 4
    q = like.new_empty((m, ldq), dtype=_E4M3)
    scale = like.new_empty((m, lds), dtype=torch.float32)
    return q if ldq == k else q[:, :k], scale if lds == _blocks(k) else scale[:, :_blocks(k)], ldq, lds


def _readable(t, size):
    """``t`` with rows that the products can read: unit stride, rows a multiple of 16
    bytes apart, 16-byte aligned; else a copy."""
    m, n = t.shape
    ld = t.stride(0) if m > 1 else -(-n // (16 // size)) * (16 // size)
    if (n <= 1 or t.stride(1) == 1) and ld * size % 16 == 0 and ld >= n and t.data_ptr() % 16 == 0:
        return t, ld
    ld = -(-n // (16 // size)) * (16 // size)
    c = t.new_empty((m, ld))
    c[:, :n].copy_(t)
    return c, ld


def _quantize(x, s):
    x, ldx = _matrix(x, "x")
    m, k = x.shape
    if k == 0:
        raise ValueError("x has no columns")
    q, scale, ldq, lds = _new_rows(m, k, x)
    _lib.check(_lib.lib().aem_quantize_fp8(x.data_ptr(), _DT[x.dtype], ldx, m, k, q.data_ptr(), ldq,
                                           scale.data_ptr(), lds, s), "aem_quantize_fp8")
    return Fp8Rows.__new__(Fp8Rows)._set(q, scale)


def quantize_fp8(x, stream=None):
    """``Fp8Rows`` of ``x [M, K]`` (float32 or bfloat16): blocks of 128 along a row share
    ``scale = max(amax / 448, 2^-126)``, ``q = e4m3(x / scale)``.  No gradient: the
    products quantise a tensor that requires one themselves."""
    _no_gradient("quantize_fp8", x, "x")
    return _on(stream, _quantize, (x,), (x,))


def _quantize_weight(w, s):
    w = w.contiguous()  # on the call's stream, like everything that reads it
    g = 1 if w.dim() == 2 else w.shape[0]
    k, n = w.shape[-2:]
    q = w.new_empty(w.shape, dtype=_E4M3)
    scale = w.new_empty(tuple(w.shape[:-2]) + (_blocks(k), _blocks(n)), dtype=torch.float32)
    _lib.check(_lib.lib().aem_quantize_fp8_weight(w.data_ptr(), _DT[w.dtype], g, k, n, q.data_ptr(), scale.data_ptr(),
                                                  s), "aem_quantize_fp8_weight")
    return q, scale


def quantize_fp8_weight(w, stream=None):
    """``w [K, N]`` or ``[G, K, N]`` (float32 or bfloat16) -> ``(q float8_e4m3fn, scale
    float32 [(G,) ceil(K/128), ceil(N/128)])`` in blocks of 128 x 128.  No gradient."""
    _no_gradient("quantize_fp8_weight", w, "w")
    if w.dim() not in (2, 3):
        raise ValueError("w must be [K, N] or [G, K, N]")
    if w.dtype not in _DT:
        raise ValueError(f"w: unsupported dtype {w.dtype} (float32 or bfloat16)")
    return _on(stream, _quantize_weight, (w,), (w,))


class Fp8Weight:
    """Packed e4m3 weight groups: ``q [K, N]`` or ``[G, K, N]`` float8_e4m3fn and
    ``scale [(G,) ceil(K/128), ceil(N/128)]`` float32.  CUDA tensors are packed on the
    device (the call waits for it), CPU tensors through ``aem_fp8weight_pack`` onto
    ``device``."""

    def __init__(self, q, scale, device=0, stream=None):
        self.handle = None
        if q.dtype != _E4M3 or q.dim() not in (2, 3):
            raise ValueError(f"q must be [K, N] or [G, K, N] float8_e4m3fn, got {tuple(q.shape)} {q.dtype}")
        g = 1 if q.dim() == 2 else q.shape[0]
        k, n = q.shape[-2:]
        want = tuple(q.shape[:-2]) + (_blocks(k), _blocks(n))
        if scale.dtype != torch.float32 or tuple(scale.shape) != want:
            raise ValueError(f"scale must be {want} float32, got {tuple(scale.shape)} {scale.dtype}")
        if q.device.type not in ("cpu", "cuda") or scale.device != q.device:
            raise ValueError(f"q and scale must be on one CUDA device or the CPU, got {q.device} and {scale.device}")
        _no_gradient("Fp8Weight", q, "q")
        _no_gradient("Fp8Weight", scale, "scale")
        h = ctypes.c_void_p()
        if q.is_cuda:
            def pack(q, scale, s):
                q, scale = q.contiguous(), scale.contiguous()  # on the call's stream
                _lib.check(_lib.lib().aem_fp8weight_pack_device(q.data_ptr(), scale.data_ptr(), g, k, n, s,
                                                                ctypes.byref(h)), "aem_fp8weight_pack_device")
                # any stream may use the weight from here on
                torch.cuda.current_stream(q.device).synchronize()
            _on(stream, pack, (q, scale), (q, scale))
            device = q.device.index
        else:
            q, scale = q.contiguous(), scale.contiguous()
            _lib.check(_lib.lib().aem_fp8weight_pack(q.data_ptr(), scale.data_ptr(), g, k, n, device,
                                                     ctypes.byref(h)), "aem_fp8weight_pack")
        self.handle, self._scratch = h.value, {}
        self.G, self.K, self.N, self.device = g, k, n, device

    def close(self):
        if getattr(self, "handle", None):
            _lib.lib().aem_fp8weight_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _product(x, w, starts, group, transposed, relu, zero_rest, out_dtype, out, s):
    L = _lib.lib()
    k, n = (w.N, w.K) if transposed else (w.K, w.N)
    if isinstance(x, Fp8Rows):
        if x.shape[1] != k:
            raise ValueError(f"x has {x.shape[1]} columns, expected {k}")
        m, like = x.shape[0], x.q
        inputs = (x.q, x.scale)
        q, ldx = _readable(x.q, 1)
        scale, lds = _readable(x.scale, 4)
        code, px, ps = _lib.E4M3, q.data_ptr(), scale.data_ptr()
        default = torch.float32
    else:
        x, ldx = _matrix(x, "x", d=k)
        m, like = x.shape[0], x
        inputs = (x,)
        code, px, ps, lds = _DT[x.dtype], x.data_ptr(), None, 0
        default = x.dtype
    if not w.handle:
        raise ValueError("the weight is closed")
    if like.get_device() != w.device:
        raise ValueError(f"x is on {like.device}, the weight on cuda:{w.device}")
    given = out
    out, ldo = _output(out, (m, n), out_dtype or (default if out is None else out.dtype), like)
    _apart(given, *inputs)
    ws, need, keep = None, 0, None
    if ps is None:
        key = (code, m, transposed)
        need = w._scratch.get(key)
        if need is None:
            need = L.aem_fp8gemm_workspace(w.handle, code, m, transposed)
            if len(w._scratch) < 1024:
                w._scratch[key] = need
        if need:
            keep = like.new_empty(need, dtype=torch.uint8)
            ws = keep.data_ptr()
    if starts is None:
        _lib.check(L.aem_fp8gemm(w.handle, group, transposed, px, code, ldx, ps, lds, m, out.data_ptr(),
                                 _DT[out.dtype], ldo, ws, need, s), "aem_fp8gemm")
    else:
        _lib.check(L.aem_grouped_fp8gemm(w.handle, starts.data_ptr(), transposed, px, code, ldx, ps, lds, m,
                                         out.data_ptr(), _DT[out.dtype], ldo, 1 if relu else 0,
                                         1 if zero_rest else 0, ws, need, s), "aem_grouped_fp8gemm")
    return out


def _check_starts(starts, w):
    if starts.dtype != torch.int32 or tuple(starts.shape) != (w.G + 1,) or not starts.is_contiguous():
        raise ValueError(f"starts must be {w.G + 1} contiguous int32 offsets")


class _ProductFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, starts, group, out_dtype, stream):
        ctx.w, ctx.group, ctx.x_dtype = w, group, x.dtype
        ctx.save_for_backward(*(() if starts is None else (starts,)))
        return _on(stream, _product, (x, starts), (x, w, starts, group, 0, False, starts is not None, out_dtype, None))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        starts = ctx.saved_tensors[0] if ctx.saved_tensors else None
        _refuse_capture("fp8_matmul" if starts is None else "grouped_fp8_matmul")
        gx = _on(None, _product, (grad, starts), (grad, ctx.w, starts, ctx.group, 1, False, starts is not None,
                                                  ctx.x_dtype, None))
        return gx, None, None, None, None, None


def fp8_matmul(x, w, group=0, out_dtype=None, out=None, stream=None):
    """``x [M, K] @`` group ``group`` of ``w`` -> ``[M, N]``: x a float32 or bfloat16
    tensor, quantised in the call, or ``Fp8Rows``.  ``out_dtype`` (float32 or bfloat16)
    defaults to x's, for ``Fp8Rows`` to float32."""
    if not isinstance(x, Fp8Rows) and _differentiable("fp8_matmul", out, stream, x):
        return _apply(_ProductFn, stream, x, w, None, group, out_dtype)
    return _on(stream, _product, (x, out), (x, w, None, group, 0, False, False, out_dtype, out))


def fp8_matmul_backward(grad_out, w, group=0, out_dtype=None, out=None, stream=None):
    """Gradient of ``fp8_matmul`` with respect to x: ``grad_out [M, N]`` (a tensor,
    quantised in the call, or ``Fp8Rows``) times the transposed weight -> ``[M, K]``."""
    if not isinstance(grad_out, Fp8Rows):
        _no_tangent("fp8_matmul_backward", grad_out)
    return _on(stream, _product, (grad_out, out), (grad_out, w, None, group, 1, False, False, out_dtype, out))


def grouped_fp8_matmul(x, w, starts, relu=False, out_dtype=None, out=None, stream=None):
    """Rows ``[starts[g], starts[g+1])`` of ``x [M, K]`` (as ``fp8_matmul``) times group
    ``g`` of ``w``, for every group, with an optional ReLU.  Rows outside every group
    are not written (uninitialised where ``out`` is not given); where x requires a
    gradient they are zero, and so are their gradients."""
    _check_starts(starts, w)
    if not isinstance(x, Fp8Rows) and _differentiable("grouped_fp8_matmul", out, stream, x):
        if relu:
            raise RuntimeError("grouped_fp8_matmul: relu=True has no gradient: apply torch.relu to the product")
        return _apply(_ProductFn, stream, x, w, starts, 0, out_dtype)
    return _on(stream, _product, (x, starts, out), (x, w, starts, 0, 0, relu, False, out_dtype, out))


def grouped_fp8_matmul_backward(grad_out, w, starts, out_dtype=None, out=None, stream=None):
    """Gradient of ``grouped_fp8_matmul`` (without its ReLU) with respect to x.  Rows
    outside every group are zero."""
    _check_starts(starts, w)
    if not isinstance(grad_out, Fp8Rows):
        _no_tangent("grouped_fp8_matmul_backward", grad_out)
    return _on(stream, _product, (grad_out, starts, out), (grad_out, w, starts, 0, 1, False, True, out_dtype, out))
