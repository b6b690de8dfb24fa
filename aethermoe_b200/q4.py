"""4-bit weights with group scales: quantisation, the packed weight, and the
products of a decoding step's rows with it, dense and grouped by expert.

    q, s = quantize_q4(w, 128)                   # w [K, N] or [G, K, N]
    weight = Q4Weight(q, s, 128)                 # packed once, about K*N/2 bytes a group
    y = q4_matmul(x, weight)                     # x [M, K]
    h = grouped_q4_matmul(rows, weight, order.starts, relu=True)

Tensors are torch CUDA tensors; every kernel is in ``libaethermoe.so``
(``aem_quantize_q4`` and the following calls of ``include/aem.h``, which
define the results).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .dispatch import _DT, _apart, _matrix, _no_tangent, _on, _output


def _no_gradient(what, x, name="x"):
    _no_tangent(what, x)
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no gradient: detach {name} or call it under torch.no_grad()")


def _quantize(w, group_size, scale_dtype, s):
    w = w.contiguous()  # on the call's stream, like everything that reads it
    g = 1 if w.dim() == 2 else w.shape[0]
    k, n = w.shape[-2:]
    kb = -(-k // group_size)
    q = w.new_empty(w.shape, dtype=torch.int8)
    scale = w.new_empty((kb, n) if w.dim() == 2 else (g, kb, n), dtype=scale_dtype)
    _lib.check(_lib.lib().aem_quantize_q4(w.data_ptr(), _DT[w.dtype], g, k, n, group_size,
                                          q.data_ptr(), scale.data_ptr(), _DT[scale_dtype], s),
               "aem_quantize_q4")
    return q, scale


def quantize_q4(w, group_size=128, scale_dtype=torch.float32, stream=None):
    """``w [K, N]`` or ``[G, K, N]`` (float32 or bfloat16) -> ``(q int8, scale)`` with
    ``scale [(G,) ceil(K/group_size), N]``: symmetric, values in [-7, 7], the
    ``group_size`` (32, 64, 128) consecutive k of a column sharing a scale.  No gradient."""
    _no_gradient("quantize_q4", w, "w")
    if w.dim() not in (2, 3):
        raise ValueError("w must be [K, N] or [G, K, N]")
    if w.dtype not in _DT or scale_dtype not in _DT:
        raise ValueError(f"unsupported dtype {w.dtype} / {scale_dtype} (float32 or bfloat16)")
    if group_size not in (32, 64, 128):
        raise ValueError(f"group_size={group_size} is not 32, 64 or 128")
    return _on(stream, _quantize, (w,), (w, group_size, scale_dtype))


class Q4Weight:
    """Packed 4-bit weight groups: ``q [K, N]`` or ``[G, K, N]`` int8 with values in
    [-7, 7] and ``scale [(G,) ceil(K/group_size), N]`` (float32 or bfloat16).
    CUDA tensors are packed on the device (the call waits for it and raises on
    a value out of range), CPU tensors and NumPy arrays through
    ``aem_q4weight_pack`` onto ``device``."""

    def __init__(self, q, scale, group_size, device=0, stream=None):
        self.handle = None
        q, scale = torch.as_tensor(q), torch.as_tensor(scale)
        if q.dtype != torch.int8 or q.dim() not in (2, 3):
            raise ValueError(f"q must be [K, N] or [G, K, N] int8, got {tuple(q.shape)} {q.dtype}")
        if scale.dtype not in _DT:
            raise ValueError(f"scale: unsupported dtype {scale.dtype} (float32 or bfloat16)")
        if group_size not in (32, 64, 128):
            raise ValueError(f"group_size={group_size} is not 32, 64 or 128")
        g = 1 if q.dim() == 2 else q.shape[0]
        k, n = q.shape[-2:]
        want = tuple(q.shape[:-2]) + (-(-k // group_size), n)
        if tuple(scale.shape) != want:
            raise ValueError(f"scale must be {want}, got {tuple(scale.shape)}")
        if q.device.type not in ("cpu", "cuda") or scale.device != q.device:
            raise ValueError(f"q and scale must be on one CUDA device or the CPU, got {q.device} and {scale.device}")
        h = ctypes.c_void_p()
        if q.is_cuda:
            def pack(q, scale, s):
                q, scale = q.contiguous(), scale.contiguous()  # on the call's stream
                st = _lib.lib().aem_q4weight_pack_checked(q.data_ptr(), scale.data_ptr(), _DT[scale.dtype], g,
                                                          k, n, group_size, s, ctypes.byref(h))
                _lib.check(st, "aem_q4weight_pack_checked")
            _on(stream, pack, (q, scale), (q, scale))
            device = q.device.index
        else:
            q, scale = q.contiguous(), scale.contiguous()
            _lib.check(_lib.lib().aem_q4weight_pack(q.data_ptr(), scale.data_ptr(), _DT[scale.dtype], g,
                                                    k, n, group_size, device, ctypes.byref(h)),
                       "aem_q4weight_pack")
        self.handle, self._scratch = h.value, {}
        self.G, self.K, self.N, self.group_size, self.device = g, k, n, group_size, device

    def close(self):
        if getattr(self, "handle", None):
            _lib.lib().aem_q4weight_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _check_weight(w, device):
    if not w.handle:
        raise ValueError("the weight is closed")
    if device.index != w.device:
        raise ValueError(f"x is on {device}, the weight on cuda:{w.device}")


def _scratch(x, w, grouped):
    """``(pointer, bytes, tensor)`` of a product's scratch."""
    key = (x.dtype, x.shape[0], grouped)
    n = w._scratch.get(key)
    if n is None:
        n = _lib.lib().aem_q4gemm_workspace(w.handle, _DT[x.dtype], x.shape[0], grouped)
        if len(w._scratch) < 1024:
            w._scratch[key] = n
    if not n:
        return None, 0, None
    t = x.new_empty(n, dtype=torch.uint8)
    return t.data_ptr(), n, t


def _matmul(x, w, group, out_dtype, out, s):
    x, ldx = _matrix(x, "x", d=w.K)
    _check_weight(w, x.device)
    m = x.shape[0]
    given = out
    out, ldo = _output(out, (m, w.N), out_dtype or (x.dtype if out is None else out.dtype), x)
    _apart(given, x)
    ws, n, keep = _scratch(x, w, 0)
    _lib.check(_lib.lib().aem_q4gemm(w.handle, group, x.data_ptr(), _DT[x.dtype], ldx, m,
                                     out.data_ptr(), _DT[out.dtype], ldo, ws, n, s), "aem_q4gemm")
    return out


def _grouped(x, w, starts, relu, out_dtype, out, s):
    x, ldx = _matrix(x, "x", d=w.K)
    _check_weight(w, x.device)
    if starts.dtype != torch.int32 or tuple(starts.shape) != (w.G + 1,) or not starts.is_contiguous():
        raise ValueError(f"starts must be {w.G + 1} contiguous int32 offsets")
    m = x.shape[0]
    given = out
    out, ldo = _output(out, (m, w.N), out_dtype or (x.dtype if out is None else out.dtype), x)
    _apart(given, x)
    ws, n, keep = _scratch(x, w, 1)
    _lib.check(_lib.lib().aem_grouped_q4gemm(w.handle, starts.data_ptr(), x.data_ptr(), _DT[x.dtype],
                                             ldx, m, out.data_ptr(), _DT[out.dtype], ldo,
                                             1 if relu else 0, ws, n, s), "aem_grouped_q4gemm")
    return out


def q4_matmul(x, w, group=0, out_dtype=None, out=None, stream=None):
    """``x [M, K] @`` group ``group`` of ``w`` -> ``[M, N]`` (``out_dtype`` defaults to
    x's): the weight stream of a decoding step.  For inference: no gradient."""
    _no_gradient("q4_matmul", x)
    return _on(stream, _matmul, (x, out), (x, w, group, out_dtype, out))


def grouped_q4_matmul(x, w, starts, relu=False, out_dtype=None, out=None, stream=None):
    """Rows ``[starts[g], starts[g+1])`` of ``x [M, K]`` times group ``g`` of ``w``,
    for every group, with an optional ReLU.  Rows outside every group are not
    written (uninitialised where ``out`` is not given).  For inference: no gradient."""
    _no_gradient("grouped_q4_matmul", x)
    return _on(stream, _grouped, (x, starts, out), (x, w, starts, relu, out_dtype, out))
