"""Encoder operators on B200 kernels: layer norm, linear with bias, activation and residual, and a
gated linear recurrence over time.

All take float32, bfloat16 or float16 CUDA tensors, compute in float32 and round a result once.
They are differentiable once.  Under autocast ``linear`` runs in the autocast type; the others run
in the type of their input (with float32 parameters, states and statistics).
"""

from typing import NamedTuple

import torch

from .. import _native as nat
from . import _ops

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


class GatedScanOutput(NamedTuple):
    """Result of ``gated_scan``: ``output`` [B,T,D] and the last ``state`` [B,D] (float32)."""

    output: torch.Tensor
    state: torch.Tensor


def _check_type(name, t):
    if t.dtype not in _TYPES:
        raise TypeError("{} must be float32, bfloat16 or float16, got {}".format(name, t.dtype))


def _check_device(first, *rest):
    device = first.device
    if device.type != "cuda":
        nat.require_cuda(first)
    for t in rest:
        if t is not None and t.device != device:
            nat.require_cuda(t)
            raise ValueError("all tensors must be on one device, got {} and {}".format(
                device, t.device))


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _check_parameter(name, p, x):
    if p.ndim != 1 or p.shape[0] != x.shape[-1]:
        raise ValueError("{} must have shape [{}], got {}".format(name, x.shape[-1],
                                                                  list(p.shape)))
    if p.dtype != x.dtype and p.dtype != torch.float32:
        raise TypeError("{} must be float32 or of x's type {}, got {}".format(name, x.dtype,
                                                                              p.dtype))


def layer_norm(x, weight=None, bias=None, *, eps=1e-5):
    """Layer norm over the last dimension: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    Args:
        x: [..., D] float32, bfloat16 or float16; rows may be strided.
        weight, bias: [D] of x's type or float32 (both of one type), or None.
        eps: Added to the variance (>= 0).

    Returns:
        [..., D] of x's type.
    """
    _check_type("x", x)
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError("x must have shape [..., D] with D > 0")
    if weight is not None:
        _check_parameter("weight", weight, x)
    if bias is not None:
        _check_parameter("bias", bias, x)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one type")
    if not eps >= 0:
        raise ValueError("eps must be >= 0")
    _check_device(x, weight, bias)
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if torch.compiler.is_compiling():
        return _ops.layer_norm_op(x, weight, bias, float(eps))[0]
    if _wants_grad(x, weight, bias):
        return _ops.LayerNormFunction.apply(x, weight, bias, float(eps))
    return _ops.layer_norm_forward(x, weight, bias, float(eps), False)[0]


def linear(x, weight, bias=None, *, activation=None, residual=None):
    """Linear layer with its epilogue: ``activation(x @ weight.T + bias) + residual``.

    Args:
        x: [..., K] float32, bfloat16 or float16; rows may be strided.
        weight: [N, K].
        bias: [N] or None.
        activation: None, "relu", "gelu" (with erf), "silu" or "sigmoid".
        residual: [..., N] (the result's shape) or None, added after the activation.

    All tensors have one type (under autocast they are cast to the autocast type).

    Returns:
        [..., N] of that type.  float32 products keep float32 precision.
    """
    if activation not in _ops.ACTIVATIONS:
        raise ValueError("activation must be one of {}, got {!r}".format(
            [a for a in _ops.ACTIVATIONS if a not in (None, "none")] + [None], activation))
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        x, weight, bias, residual = (None if t is None else t.to(dtype)
                                     for t in (x, weight, bias, residual))
    _check_type("x", x)
    if weight.ndim != 2 or 0 in weight.shape:
        raise ValueError("weight must have shape [N, K] with N, K > 0")
    n, k = weight.shape
    if x.ndim < 1 or x.shape[-1] != k:
        raise ValueError("x must have shape [..., {}], got {}".format(k, list(x.shape)))
    if bias is not None and (bias.ndim != 1 or bias.shape[0] != n):
        raise ValueError("bias must have shape [{}], got {}".format(n, list(bias.shape)))
    if residual is not None and residual.shape != (*x.shape[:-1], n):
        raise ValueError("residual must have shape {}, got {}".format([*x.shape[:-1], n],
                                                                      list(residual.shape)))
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError("{} must be of x's type {}, got {}".format(name, x.dtype, t.dtype))
    _check_device(x, weight, bias, residual)
    act = _ops.ACTIVATIONS[activation]
    bias = None if bias is None else bias.contiguous()
    if torch.compiler.is_compiling():
        return _ops.linear_op(x, weight, bias, residual, act)[0]
    if _wants_grad(x, weight, bias, residual):
        return _ops.LinearFunction.apply(x, weight, bias, residual, act)
    return _ops.linear_forward(x, weight, bias, residual, act, False)[0]


def gated_scan(x, gate, state=None, *, lengths=None):
    """Gated linear recurrence over time, ``f = sigmoid(gate)``::

        h_t = f_t * h_{t-1} + (1 - f_t) * x_t

    Args:
        x, gate: [B,T,D] of one type; any batch and time strides (two halves of one projection,
            for instance).
        state: [B,D] float32, the state before the first frame; None for zeros.
        lengths: [B] integers; from frame ``lengths[b]`` on a sequence keeps its state, its
            outputs are 0 and its inputs are not read (whatever they hold).

    Returns:
        GatedScanOutput(output [B,T,D] of x's type, state [B,D] float32).
    """
    _check_type("x", x)
    if x.ndim != 3 or x.shape[2] == 0:
        raise ValueError("x must have shape [batch, time, feature] with features")
    if gate.shape != x.shape:
        raise ValueError("gate must have x's shape {}, got {}".format(list(x.shape),
                                                                      list(gate.shape)))
    if gate.dtype != x.dtype:
        raise TypeError("gate must be of x's type {}, got {}".format(x.dtype, gate.dtype))
    _check_state(state, x.shape[0], x.shape[2])
    if lengths is not None:
        if lengths.shape != x.shape[:1]:
            raise ValueError("lengths must have shape [{}], got {}".format(x.shape[0],
                                                                           list(lengths.shape)))
        if lengths.dtype not in (torch.int64, torch.int32):
            raise TypeError("lengths must be int64 or int32, got {}".format(lengths.dtype))
    _check_device(x, gate, state, lengths)
    if lengths is not None:
        lengths = lengths.to(torch.int64).contiguous()
    if torch.compiler.is_compiling():
        return GatedScanOutput(*_ops.gated_scan_op(x, gate, state, lengths)[:2])
    if _wants_grad(x, gate, state):
        return GatedScanOutput(*_ops.GatedScanFunction.apply(x, gate, state, lengths))
    return GatedScanOutput(*_ops.gated_scan_forward(x, gate, state, lengths, False)[:2])


def _check_state(state, batch, dim):
    if state is None:
        return
    if state.ndim != 2 or state.shape[0] != batch or state.shape[1] != dim:
        raise ValueError("state must have shape [{}, {}], got {}".format(batch, dim,
                                                                         list(state.shape)))
    if state.dtype != torch.float32:
        raise TypeError("state must be float32, got {}".format(state.dtype))


def gated_scan_step(x, gate, state):
    """One frame of ``gated_scan`` for streams: ``state`` is updated in place.

    Args:
        x, gate: [B,D] of one type.
        state: [B,D] float32, contiguous.

    Returns:
        [B,D] of x's type.  Not differentiable.
    """
    _check_type("x", x)
    if x.ndim != 2 or x.shape[1] == 0:
        raise ValueError("x must have shape [batch, feature] with features")
    if gate.shape != x.shape:
        raise ValueError("gate must have x's shape {}, got {}".format(list(x.shape),
                                                                      list(gate.shape)))
    if gate.dtype != x.dtype:
        raise TypeError("gate must be of x's type {}, got {}".format(x.dtype, gate.dtype))
    if state is None:
        raise ValueError("state must be a [B,D] tensor: it is updated in place")
    _check_state(state, *x.shape)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    _check_device(x, gate, state)
    if _wants_grad(x, gate, state):
        raise RuntimeError("gated_scan_step is not differentiable; use gated_scan, or no_grad")
    return _ops.gated_scan_step(x, gate, state)
