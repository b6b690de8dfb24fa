"""Routing of tokens to experts from a router's logits, with its gradient.

    ids, weights = route_tokens(logits, k)                       # [T, k] int32, [T, k] float32
    ids, weights = route_tokens(logits, 8, score="sigmoid", bias=balance, groups=8, top_groups=4,
                                group_top=2, renormalize=True, scale=2.5)
    rows, order = dispatch.dispatch(x, ids, num_experts)

For callers with their own router projection: softmax or sigmoid scores, a
balance bias that takes part in the choice alone, groups of experts, top-k and
renormalised weights.  Tensors are torch CUDA tensors; the kernels are in
``libaethermoe.so`` (``aem_route_tokens`` and ``aem_route_tokens_backward`` of
``include/aem.h``, which define the results).  An id of -1 (fewer than k experts
can be chosen) is a unit without an expert for the dispatch and the combine.
``route_tokens`` takes part in autograd when the logits require a gradient; a
training step that is captured into a CUDA graph calls ``route_tokens_backward``
itself (the differentiable form refuses to be captured).  Forward-mode tangents
are refused.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .dispatch import _DT, _apart, _apply, _differentiable, _matrix, _no_tangent, _on, _output, _refuse_capture, _weights

_SCORES = {"softmax": _lib.SCORE_SOFTMAX, "sigmoid": _lib.SCORE_SIGMOID}


def _config(k, score, groups, top_groups, group_top, renormalize, scale):
    if score not in _SCORES:
        raise ValueError(f"score={score!r} is not 'softmax' or 'sigmoid'")
    c = _lib.RouteConfig(_SCORES[score], k, groups, top_groups, group_top, 1 if renormalize else 0, scale)
    if c.k != k or c.groups != groups or c.top_groups != top_groups or c.group_top != group_top:
        raise ValueError(f"k={k}, groups={groups}, top_groups={top_groups} or group_top={group_top} is out of range")
    return c


def _check_bias(bias, logits):
    if bias is None:
        return None
    if bias.dtype != torch.float32 or tuple(bias.shape) != (logits.shape[1],):
        raise ValueError(f"bias must be ({logits.shape[1]},) float32, got {tuple(bias.shape)} {bias.dtype}")
    return bias.contiguous()


def _route(logits, bias, config, s):
    logits, ld = _matrix(logits, "logits")
    bias = _check_bias(bias, logits)
    t, e = logits.shape
    ids = logits.new_empty((t, max(config.k, 0)), dtype=torch.int32)
    weights = logits.new_empty((t, max(config.k, 0)), dtype=torch.float32)
    _lib.check(_lib.lib().aem_route_tokens(ctypes.byref(config), logits.data_ptr(), _DT[logits.dtype], ld, t, e,
                                           None if bias is None else bias.data_ptr(), ids.data_ptr(),
                                           weights.data_ptr(), s), "aem_route_tokens")
    return ids, weights


def _route_backward(grad, logits, ids, config, out, s):
    logits, ld = _matrix(logits, "logits")
    t, e = logits.shape
    if ids.dtype != torch.int32 or tuple(ids.shape) != (t, config.k):
        raise ValueError(f"ids must be {(t, config.k)} int32, got {tuple(ids.shape)} {ids.dtype}")
    if config.k > 1 and ids.stride(1) != 1:
        ids = ids.contiguous()
    grad, ldg = _weights(grad, (t, config.k), "grad_weights")
    given = out
    out, ldo = _output(out, (t, e), logits.dtype, logits)
    _apart(given, logits, grad, ids)
    _lib.check(_lib.lib().aem_route_tokens_backward(
        ctypes.byref(config), grad.data_ptr(), ldg, logits.data_ptr(), _DT[logits.dtype], ld, t, e, ids.data_ptr(),
        ids.stride(0) if t > 1 else config.k, out.data_ptr(), ldo, s), "aem_route_tokens_backward")
    return out


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, config, stream):
        ids, weights = _on(stream, _route, (logits, bias), (logits, bias, config))
        ctx.save_for_backward(logits, ids)
        ctx.config = config
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return ids, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, grad):
        _refuse_capture("route_tokens")
        if grad is None:
            return None, None, None, None
        logits, ids = ctx.saved_tensors
        return _on(None, _route_backward, (grad, logits, ids), (grad, logits, ids, ctx.config, None)), None, None, None


def route_tokens(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=False,
                 scale=1.0, stream=None):
    """``(ids [T, k] int32, weights [T, k] float32)`` of ``logits [T, E]`` (float32 or
    bfloat16): the k experts of the largest ``score + bias`` (``bias [E]`` float32 or
    ``None``) in falling order, ties to the lower index, and ``scale`` times their
    scores, without the bias, divided by their sum with ``renormalize``.  With
    ``groups``, only experts of the ``top_groups`` groups of ``E / groups``
    neighbours with the largest value can be chosen; a group's value is its largest
    key or the sum of its two (``group_top``).  The bias has no gradient."""
    config = _config(k, score, groups, top_groups, group_top, renormalize, scale)
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("route_tokens: the bias has no gradient: detach it")
    if _differentiable("route_tokens", None, stream, logits):
        return _apply(_RouteFn, stream, logits, bias, config)
    _no_tangent("route_tokens", bias)
    return _on(stream, _route, (logits, bias), (logits, bias, config))


def route_tokens_backward(grad_weights, logits, ids, score="softmax", renormalize=False, scale=1.0, out=None,
                          stream=None):
    """Gradient of the weights of ``route_tokens`` with respect to the logits, ``[T, E]``
    in their dtype; ``ids`` as it returned them.  Bias and groups only chose the ids."""
    _no_tangent("route_tokens_backward", grad_weights, logits)
    if ids.dim() != 2:
        raise ValueError(f"ids must be [T, k] int32, got {tuple(ids.shape)} {ids.dtype}")
    config = _config(ids.shape[1], score, 1, 1, 1, renormalize, scale)
    return _on(stream, _route_backward, (grad_weights, logits, ids, out), (grad_weights, logits, ids, config, out))
