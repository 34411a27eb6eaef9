"""The encoder operators as torch custom ops, for ``torch.compile``, tracers and transforms.

Eager calls go straight to the host extension (``csrc/host/encoder_host.cpp``), which checks the
arguments, allocates, records autograd and calls the C ABI.  ``torch.compile`` needs ops it can
trace: ``torchwarp_b200::layer_norm``, ``linear``, ``gated_scan`` with fakes and registered
backwards, and ``gated_scan_step``, over the same extension.  The extension itself calls them where
a tracer, a dispatch mode, a transform or a tensor subclass has to see the operator.  Ops and fakes make the extension's checks of an eager call, so
a bad argument is refused while a function is traced.  ``save``: a backward will follow, and the
results that it needs are not left empty.  Backward passes are first order only.
"""

from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _native as nat

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}


# -------------------------------------------------------------- layer norm

@torch.library.custom_op("torchwarp_b200::layer_norm", mutates_args=())
def layer_norm(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor],
               eps: float, save: bool = True) -> Tuple[Tensor, Tensor]:
    y, stats = nat.host().layer_norm_forward(x, weight, bias, eps, save)
    return y, stats if save else x.new_empty((2, 0), dtype=torch.float32)


@layer_norm.register_fake
def _(x, weight, bias, eps, save=True):
    nat.host().check_layer_norm(x, weight, bias, eps)
    return (x.new_empty(x.shape),
            x.new_empty((2, x.numel() // x.shape[-1] if save else 0), dtype=torch.float32))


@torch.library.custom_op("torchwarp_b200::layer_norm_backward", mutates_args=())
def layer_norm_backward(dy: Tensor, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor],
                        stats: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    return nat.host().layer_norm_backward(dy, x, weight, bias, stats)


@layer_norm_backward.register_fake
def _(dy, x, weight, bias, stats):
    nat.host().check_layer_norm_backward(dy, x, weight, bias, stats)
    like = weight if weight is not None else bias if bias is not None else x
    return x.new_empty(x.shape), like.new_empty(x.shape[-1]), like.new_empty(x.shape[-1])


def _layer_norm_setup(ctx, inputs, output):
    x, weight, bias, _, _ = inputs
    ctx.save_for_backward(x, weight, bias, output[1])


def _layer_norm_bwd(ctx, dy, _stats):
    x, weight, bias, stats = ctx.saved_tensors
    dx, dw, db = layer_norm_backward(dy, x, weight, bias, stats)
    return dx, None if weight is None else dw, None if bias is None else db, None, None


layer_norm.register_autograd(_layer_norm_bwd, setup_context=_layer_norm_setup)


# ------------------------------------------------------------------ linear

@torch.library.custom_op("torchwarp_b200::linear", mutates_args=())
def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor],
           act: int, save: bool = True) -> Tuple[Tensor, Tensor]:
    y, z = nat.host().linear_forward(x, weight, bias, residual, act, save)
    return y, z if z is not None else x.new_empty(0)


@linear.register_fake
def _(x, weight, bias, residual, act, save=True):
    nat.host().check_linear(x, weight, bias, residual)
    n, k = weight.shape
    return (x.new_empty((*x.shape[:-1], n)),
            x.new_empty((x.numel() // k, n) if act and save else (0,)))


@torch.library.custom_op("torchwarp_b200::linear_backward", mutates_args=())
def linear_backward(dy: Tensor, x: Tensor, weight: Tensor, z: Tensor,
                    act: int) -> Tuple[Tensor, Tensor, Tensor]:
    return nat.host().linear_backward(dy, x, weight, z if act else None, act)


@linear_backward.register_fake
def _(dy, x, weight, z, act):
    nat.host().check_linear_backward(dy, x, weight, z if act else None, act)
    return (x.new_empty(x.shape), weight.new_empty(weight.shape),
            weight.new_empty(weight.shape[0]))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, residual, act, _ = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.has = (bias is not None, residual is not None)
    ctx.act = act


def _linear_bwd(ctx, dy, _z):
    x, weight, z = ctx.saved_tensors
    dx, dw, db = linear_backward(dy, x, weight, z, ctx.act)
    return dx, dw, db if ctx.has[0] else None, dy if ctx.has[1] else None, None, None


linear.register_autograd(_linear_bwd, setup_context=_linear_setup)


# -------------------------------------------------------------- gated scan

@torch.library.custom_op("torchwarp_b200::gated_scan", mutates_args=())
def gated_scan(x: Tensor, gate: Tensor, h0: Optional[Tensor],
               lengths: Optional[Tensor], save: bool = True) -> Tuple[Tensor, Tensor, Tensor]:
    y, state, carry = nat.host().gated_scan_forward(x, gate, h0, lengths, save)
    return y, state, carry if save else x.new_empty(0, dtype=torch.uint8)


@gated_scan.register_fake
def _(x, gate, h0, lengths, save=True):
    nat.host().check_gated_scan(x, gate, h0, lengths)
    b, t, d = x.shape
    frames = 8 if x.element_size() == 4 else 16  # of a run, whose state is saved; sizes may be symbols
    states = 4 * b * d * ((t + frames - 1) // frames) if save else 0
    return (x.new_empty((b, t, d)), x.new_empty((b, d), dtype=torch.float32),
            x.new_empty((states + 15) // 16 * 16, dtype=torch.uint8))


@torch.library.custom_op("torchwarp_b200::gated_scan_backward", mutates_args=())
def gated_scan_backward(dy: Optional[Tensor], dstate: Optional[Tensor], x: Tensor, gate: Tensor,
                        lengths: Optional[Tensor],
                        carry: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    return nat.host().gated_scan_backward(dy, dstate, x, gate, lengths, carry)


@gated_scan_backward.register_fake
def _(dy, dstate, x, gate, lengths, carry):
    nat.host().check_gated_scan_backward(dy, dstate, x, gate, lengths, carry)
    b, t, d = x.shape
    return (x.new_empty((b, t, d)), x.new_empty((b, t, d)),
            x.new_empty((b, d), dtype=torch.float32))


def _gated_scan_setup(ctx, inputs, output):
    x, gate, h0, lengths, _ = inputs
    ctx.save_for_backward(x, gate, lengths, output[2])
    ctx.has_h0 = h0 is not None


def _gated_scan_bwd(ctx, dy, dstate, _carry):
    x, gate, lengths, carry = ctx.saved_tensors
    dx, dgate, dh0 = gated_scan_backward(dy, dstate, x, gate, lengths, carry)
    return dx, dgate, dh0 if ctx.has_h0 else None, None, None


gated_scan.register_autograd(_gated_scan_bwd, setup_context=_gated_scan_setup)


@torch.library.custom_op("torchwarp_b200::gated_scan_step", mutates_args=("state",))
def gated_scan_step(x: Tensor, gate: Tensor, state: Tensor) -> Tensor:
    return nat.host().gated_scan_step_forward(x, gate, state)


@gated_scan_step.register_fake
def _(x, gate, state):
    nat.host().check_gated_scan_step(x, gate, state)
    return x.new_empty(x.shape)
