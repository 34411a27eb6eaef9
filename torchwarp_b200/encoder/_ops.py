"""The encoder operators over the native C ABI.

Each operator has one implementation (``*_forward`` / ``*_backward``: allocate the outputs, call
the C entry) behind two front ends:

* an autograd Function, for eager calls, where the host's time is the call's time;
* custom ops ``torchwarp_b200::layer_norm``, ``linear`` and ``gated_scan`` with fakes and
  registered backwards, for ``torch.compile``.

Backward passes are first order only: differentiating one raises.
"""

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import _native as nat

# [m, n] products of up to this many rows take no workspace (csrc/linear.cu)
_SMALL_ROWS = 8


def _first_order(fn):
    """torch's ``once_differentiable``, at no cost to a backward that records no graph."""
    guarded = once_differentiable(fn)

    def backward(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else fn)(ctx, *grads)

    return backward


ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}


def rows_of(x):
    """``x`` as (tensor, row stride) with the last dimension contiguous: a view where the leading
    dimensions collapse, else a copy."""
    if x.is_contiguous():
        return x, x.shape[-1]
    x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 and x.shape[1] != 1:
        x = x.contiguous()
    return x, x.stride(0)


def frames_of(x):
    """[B, T, D] with the last dimension contiguous."""
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _dense_like(x):
    """An uninitialised contiguous tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else \
        torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _p(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# -------------------------------------------------------------- layer norm

def _mean_rstd(stats, rows):
    """Pointers to the two rows of ``stats`` [2, rows]: means, then 1 / standard deviations."""
    if stats is None:
        return None, None
    at = stats.data_ptr()
    return at, at + 4 * rows


def layer_norm_forward(x, weight, bias, eps, save):
    d = x.shape[-1]
    rows = x.numel() // d
    y = _dense_like(x)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if save else None
    if rows:
        xr, stride = rows_of(x)
        param = weight if weight is not None else bias
        nat.launch("layer_norm_forward", nat.entry("tw_layer_norm_forward", x.dtype), x.device,
                   xr.data_ptr(), stride, _p(weight), _p(bias),
                   int(param is not None and param.dtype != x.dtype), rows, d, eps, y.data_ptr(),
                   *_mean_rstd(stats, rows))
    return y, stats


def layer_norm_backward(dy, x, weight, bias_dtype, stats, need):
    """(dx, dweight, dbias), each only where `need` says so."""
    d = x.shape[-1]
    rows = x.numel() // d
    ptype = weight.dtype if weight is not None else bias_dtype or x.dtype
    dx = _dense_like(x) if need[0] else None
    dw = torch.empty(d, dtype=ptype, device=x.device) if need[1] else None
    db = torch.empty(d, dtype=ptype, device=x.device) if need[2] else None
    if any(need):
        if dy.dtype != x.dtype:
            dy = dy.to(x.dtype)
        (xr, xs), (gr, gs) = rows_of(x), rows_of(dy)
        nbytes = nat.lib().tw_layer_norm_workspace_bytes(rows, d)
        ws = _workspace(nbytes, x.device)
        nat.launch("layer_norm_backward", nat.entry("tw_layer_norm_backward", x.dtype), x.device,
                   gr.data_ptr(), gs, xr.data_ptr(), xs, _p(weight), int(ptype != x.dtype),
                   *_mean_rstd(stats, rows), rows, d, _p(dx), _p(dw), _p(db), _p(ws),
                   nbytes)
    return dx, dw, db


class LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = layer_norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        return (*layer_norm_backward(dy, x, weight, ctx.bias_dtype, stats,
                                     ctx.needs_input_grad[:3]), None)


@torch.library.custom_op("torchwarp_b200::layer_norm", mutates_args=())
def layer_norm_op(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor],
                  eps: float) -> Tuple[Tensor, Tensor]:
    return layer_norm_forward(x, weight, bias, eps, True)


@layer_norm_op.register_fake
def _(x, weight, bias, eps):
    return (x.new_empty(x.shape),
            x.new_empty((2, x.numel() // x.shape[-1]), dtype=torch.float32))


@torch.library.custom_op("torchwarp_b200::layer_norm_backward", mutates_args=())
def layer_norm_backward_op(dy: Tensor, x: Tensor, weight: Optional[Tensor],
                           param: Optional[Tensor],
                           stats: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    return layer_norm_backward(dy, x, weight, None if param is None else param.dtype, stats,
                               (True, True, True))


@layer_norm_backward_op.register_fake
def _(dy, x, weight, param, stats):
    like = weight if weight is not None else param if param is not None else x
    return (x.new_empty(x.shape), like.new_empty(x.shape[-1]), like.new_empty(x.shape[-1]))


def _layer_norm_setup(ctx, inputs, output):
    x, weight, bias, _ = inputs
    ctx.save_for_backward(x, weight, bias, output[1])


def _layer_norm_bwd(ctx, dy, _stats):
    x, weight, bias, stats = ctx.saved_tensors
    dx, dw, db = layer_norm_backward_op(dy, x, weight, bias, stats)
    return dx, None if weight is None else dw, None if bias is None else db, None


layer_norm_op.register_autograd(_layer_norm_bwd, setup_context=_layer_norm_setup)


# ------------------------------------------------------------------ linear

def _unaligned(a, stride_a, b, stride_b):
    """1 when a row of 16-bit elements may start off a 16-byte boundary."""
    return int((a.data_ptr() | b.data_ptr()) & 15 != 0 or (stride_a | stride_b) & 7 != 0
               or stride_a < a.shape[-1] or stride_b < b.shape[-1])


def linear_forward(x, weight, bias, residual, act, save):
    n, k = weight.shape
    m = x.numel() // k
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    z = torch.empty((m, n), dtype=x.dtype, device=x.device) if save and act else None
    if m:
        (xr, xs), (wr, wst) = rows_of(x), rows_of(weight)
        rr, rs = (None, 0) if residual is None else rows_of(residual)
        nbytes = 0
        if m > _SMALL_ROWS:
            nbytes = nat.lib().tw_linear_workspace_bytes(m, n, k, x.element_size(), act, 0,
                                                         _unaligned(xr, xs, wr, wst))
        ws = _workspace(nbytes, x.device)
        nat.launch("linear_forward", nat.entry("tw_linear_forward", x.dtype), x.device,
                   xr.data_ptr(), xs, wr.data_ptr(), wst,
                   None if bias is None else bias.data_ptr(), _p(rr), rs, m, n, k, act,
                   y.data_ptr(), _p(z), _p(ws), nbytes)
    return y, z


def linear_backward(dy, x, weight, z, act, need):
    """(dx, dweight, dbias), each only where `need` says so."""
    n, k = weight.shape
    m = x.numel() // k
    dev = x.device
    dx = _dense_like(x) if need[0] else None
    dw = _dense_like(weight) if need[1] else None
    db = torch.empty(n, dtype=x.dtype, device=dev) if need[2] else None
    if any(need):
        if dy.dtype != x.dtype:
            dy = dy.to(x.dtype)
        (gr, gs), (xr, xs), (wr, wst) = rows_of(dy), rows_of(x), rows_of(weight)
        nbytes = nat.lib().tw_linear_workspace_bytes(
            m, n, k, x.element_size(), act, 1,
            _unaligned(xr, xs, wr, wst) or _unaligned(gr, gs, gr, gs))
        ws = _workspace(nbytes, dev)
        nat.launch("linear_backward", nat.entry("tw_linear_backward", x.dtype), dev,
                   gr.data_ptr(), gs, xr.data_ptr(), xs, wr.data_ptr(), wst, _p(z), m, n, k, act,
                   _p(dx), _p(dw), _p(db), _p(ws), nbytes)
    return dx, dw, db


class LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, z = linear_forward(x, weight, bias, residual, act, True)
        ctx.save_for_backward(x, weight, z)
        ctx.act = act
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*linear_backward(dy, x, weight, z, ctx.act, need[:3]),
                dy if need[3] else None, None)


@torch.library.custom_op("torchwarp_b200::linear", mutates_args=())
def linear_op(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor],
              act: int) -> Tuple[Tensor, Tensor]:
    y, z = linear_forward(x, weight, bias, residual, act, True)
    return y, z if z is not None else x.new_empty(0)


@linear_op.register_fake
def _(x, weight, bias, residual, act):
    n, k = weight.shape
    return (x.new_empty((*x.shape[:-1], n)),
            x.new_empty((x.numel() // k, n) if act else (0,)))


@torch.library.custom_op("torchwarp_b200::linear_backward", mutates_args=())
def linear_backward_op(dy: Tensor, x: Tensor, weight: Tensor, z: Tensor,
                       act: int) -> Tuple[Tensor, Tensor, Tensor]:
    return linear_backward(dy, x, weight, z if act else None, act, (True, True, True))


@linear_backward_op.register_fake
def _(dy, x, weight, z, act):
    return (x.new_empty(x.shape), weight.new_empty(weight.shape),
            weight.new_empty(weight.shape[0]))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, residual, act = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.has = (bias is not None, residual is not None)
    ctx.act = act


def _linear_bwd(ctx, dy, _z):
    x, weight, z = ctx.saved_tensors
    dx, dw, db = linear_backward_op(dy, x, weight, z, ctx.act)
    return dx, dw, db if ctx.has[0] else None, dy if ctx.has[1] else None, None


linear_op.register_autograd(_linear_bwd, setup_context=_linear_setup)


# -------------------------------------------------------------- gated scan

def gated_scan_forward(x, gate, h0, lengths, save):
    b, t, d = x.shape
    y = _dense_like(x)
    state = torch.empty((b, d), dtype=torch.float32, device=x.device)
    carry = None
    nbytes = 0
    if save:
        nbytes = nat.lib().tw_gated_scan_carry_bytes(b, t, d)
        carry = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    if b:
        x, gate = frames_of(x), frames_of(gate)
        h0 = None if h0 is None else h0.contiguous()
        nat.launch("gated_scan_forward", nat.entry("tw_gated_scan_forward", x.dtype), x.device,
                   x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0),
                   gate.stride(1), _p(h0), _p(lengths), b, t, d, y.data_ptr(), state.data_ptr(),
                   _p(carry), nbytes)
    return y, state, carry


def gated_scan_backward(dy, dstate, x, gate, lengths, carry):
    """(dx, dgate, dh0) for dL/dy and dL/dstate (either may be None)."""
    b, t, d = x.shape
    dx, dgate = _dense_like(x), _dense_like(x)
    dh0 = torch.empty((b, d), dtype=torch.float32, device=x.device)
    if b:
        x, gate = frames_of(x), frames_of(gate)
        dy = torch.zeros_like(dx) if dy is None else frames_of(dy.to(x.dtype))
        dstate = None if dstate is None else dstate.float().contiguous()
        nat.launch("gated_scan_backward", nat.entry("tw_gated_scan_backward", x.dtype), x.device,
                   dy.data_ptr(), dy.stride(0), dy.stride(1), _p(dstate), x.data_ptr(),
                   x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1),
                   _p(lengths), carry.data_ptr(), carry.numel(), b, t, d, dx.data_ptr(),
                   dgate.data_ptr(), dh0.data_ptr())
    return dx, dgate, dh0


class GatedScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lengths):
        y, state, carry = gated_scan_forward(x, gate, h0, lengths, True)
        ctx.save_for_backward(x, gate, lengths, carry)
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @_first_order
    def backward(ctx, dy, dstate):
        if dy is None and dstate is None:
            return None, None, None, None
        x, gate, lengths, carry = ctx.saved_tensors
        dx, dgate, dh0 = gated_scan_backward(dy, dstate, x, gate, lengths, carry)
        return dx, dgate, dh0 if ctx.needs_input_grad[2] else None, None


@torch.library.custom_op("torchwarp_b200::gated_scan", mutates_args=())
def gated_scan_op(x: Tensor, gate: Tensor, h0: Optional[Tensor],
                  lengths: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    return gated_scan_forward(x, gate, h0, lengths, True)


@gated_scan_op.register_fake
def _(x, gate, h0, lengths):
    b, t, d = x.shape
    return (x.new_empty((b, t, d)), x.new_empty((b, d), dtype=torch.float32),
            x.new_empty(nat.lib().tw_gated_scan_carry_bytes(b, t, d), dtype=torch.uint8))


@torch.library.custom_op("torchwarp_b200::gated_scan_backward", mutates_args=())
def gated_scan_backward_op(dy: Optional[Tensor], dstate: Optional[Tensor], x: Tensor, gate: Tensor,
                           lengths: Optional[Tensor],
                           carry: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    return gated_scan_backward(dy, dstate, x, gate, lengths, carry)


@gated_scan_backward_op.register_fake
def _(dy, dstate, x, gate, lengths, carry):
    b, t, d = x.shape
    return (x.new_empty((b, t, d)), x.new_empty((b, t, d)),
            x.new_empty((b, d), dtype=torch.float32))


def _gated_scan_setup(ctx, inputs, output):
    x, gate, h0, lengths = inputs
    ctx.save_for_backward(x, gate, lengths, output[2])
    ctx.has_h0 = h0 is not None


def _gated_scan_bwd(ctx, dy, dstate, _carry):
    x, gate, lengths, carry = ctx.saved_tensors
    dx, dgate, dh0 = gated_scan_backward_op(dy, dstate, x, gate, lengths, carry)
    return dx, dgate, dh0 if ctx.has_h0 else None, None


gated_scan_op.register_autograd(_gated_scan_bwd, setup_context=_gated_scan_setup)


def gated_scan_step(x, gate, state):
    b, d = x.shape
    y = _dense_like(x)
    if b:
        (xr, xs), (gr, gs) = rows_of(x), rows_of(gate)
        nat.launch("gated_scan_step", nat.entry("tw_gated_scan_step", x.dtype), x.device,
                   xr.data_ptr(), xs, gr.data_ptr(), gs, state.data_ptr(), b, d, y.data_ptr())
        torch.autograd.graph.increment_version(state)
    return y
