"""Encoder operators on B200 kernels: layer norm, linear with bias, activation and residual, and a
gated linear recurrence over time.

All take float32, bfloat16 or float16 CUDA tensors, compute in float32 and round a result once.
They are differentiable once, in reverse mode (a forward-mode tangent is refused).  Under autocast ``linear`` runs in the autocast type; the others run
in the type of their input (with float32 parameters, states and statistics).
"""

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .. import _native as nat
from . import _ops


@torch.compiler.assume_constant_result
def _forward_mode():
    return forward_ad._current_level >= 0


def _compiling():
    """Whether a call is being traced by torch.compile, where it becomes a custom op.  An op does
    not see the tangents of what it is traced with: forward mode is refused there as a whole."""
    if not torch.compiler.is_compiling():
        return False
    if _forward_mode():
        raise RuntimeError("the encoder operators have no forward-mode derivative; their backward "
                           "is first order")
    return True


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class GatedScanOutput(NamedTuple):
    """Result of ``gated_scan``: ``output`` [B,T,D] and the last ``state`` [B,D] (float32)."""

    output: torch.Tensor
    state: torch.Tensor


def layer_norm(x, weight=None, bias=None, *, eps=1e-5):
    """Layer norm over the last dimension: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    Args:
        x: [..., D] float32, bfloat16 or float16; rows may be strided and may overlap.
        weight, bias: [D] of x's type or float32 (both of one type), or None.
        eps: Added to the variance (>= 0).

    Returns:
        [..., D] of x's type.
    """
    if _compiling():
        return _ops.layer_norm(x, weight, bias, float(eps), _wants_grad(x, weight, bias))[0]
    return nat.host().layer_norm(x, weight, bias, eps)


def linear(x, weight, bias=None, *, activation=None, residual=None):
    """Linear layer with its epilogue: ``activation(x @ weight.T + bias) + residual``.

    Args:
        x: [..., K] float32, bfloat16 or float16; rows may be strided.
        weight: [N, K].
        bias: [N] or None.
        activation: None, "relu", "gelu" (with erf), "silu" or "sigmoid".
        residual: [..., N] (the result's shape) or None, added after the activation.

    All tensors have one type (under autocast float32 and 16-bit ones are cast to its type).

    Returns:
        [..., N] of that type.  float32 products keep float32 precision.
    """
    if activation not in _ops.ACTIVATIONS:
        raise ValueError("activation must be one of {}, got {!r}".format(
            [a for a in _ops.ACTIVATIONS if a not in (None, "none")] + [None], activation))
    act = _ops.ACTIVATIONS[activation]
    if _compiling():
        if torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
            x, weight, bias, residual = (
                t.to(dtype) if t is not None and t.is_floating_point() and t.dtype != torch.float64
                else t for t in (x, weight, bias, residual))
        return _ops.linear(x, weight, bias, residual, act,
                           _wants_grad(x, weight, bias, residual))[0]
    return nat.host().linear(x, weight, bias, residual, act)


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
    if _compiling():
        return GatedScanOutput(*_ops.gated_scan(x, gate, state, lengths,
                                                 _wants_grad(x, gate, state))[:2])
    return GatedScanOutput(*nat.host().gated_scan(x, gate, state, lengths))


def gated_scan_step(x, gate, state):
    """One frame of ``gated_scan`` for streams: ``state`` is updated in place.

    Args:
        x, gate: [B,D] of one type.
        state: [B,D] float32, contiguous.

    Returns:
        [B,D] of x's type.  Not differentiable.
    """
    if _compiling():
        if _wants_grad(x, gate, state):
            raise RuntimeError("gated_scan_step is not differentiable; use gated_scan, or no_grad")
        return _ops.gated_scan_step(x, gate, state)
    return nat.host().gated_scan_step(x, gate, state)
