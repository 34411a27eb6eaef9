"""``nn.Module`` front ends of the encoder operators."""

import math

import torch
import torch.nn as nn

from . import _ops
from .functional import gated_scan, gated_scan_step, layer_norm, linear


class LayerNorm(nn.Module):
    """Layer norm over the last dimension; see ``torchwarp_b200.functional.layer_norm``."""

    def __init__(self, dim, eps=1e-5, *, device=None, dtype=None):
        super().__init__()
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, eps=self.eps)

    def extra_repr(self):
        return "{}, eps={}".format(self.weight.shape[0], self.eps)


class Linear(nn.Module):
    """Linear layer with its activation and residual; see ``torchwarp_b200.functional.linear``."""

    def __init__(self, in_features, out_features, bias=True, *, activation=None, device=None,
                 dtype=None):
        super().__init__()
        if activation not in _ops.ACTIVATIONS:
            raise ValueError("unknown activation {!r}".format(activation))
        self.activation = activation
        bound = 1.0 / math.sqrt(in_features)
        self.weight = nn.Parameter(torch.empty(out_features, in_features, device=device,
                                               dtype=dtype).uniform_(-bound, bound))
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) \
            if bias else None

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, activation=self.activation, residual=residual)

    def extra_repr(self):
        n, k = self.weight.shape
        return "{}, {}, bias={}, activation={!r}".format(k, n, self.bias is not None,
                                                         self.activation)


class EncoderBlock(nn.Module):
    """A gated recurrence over time and a two-layer map over features, each behind a layer norm
    and with a residual.

    Forward: x [B,T,D], state [B,D] float32 or None, lengths [B] or None -> (x, state).
    ``step``: one frame [B,D] with its state, updated in place.
    """

    def __init__(self, dim, hidden=None, *, device=None, dtype=None):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        hidden = 4 * dim if hidden is None else hidden
        self.norm1 = LayerNorm(dim, **kw)
        self.inner = Linear(dim, 2 * dim, **kw)
        self.outer = Linear(dim, dim, **kw)
        self.norm2 = LayerNorm(dim, **kw)
        self.up = Linear(dim, hidden, activation="gelu", **kw)
        self.down = Linear(hidden, dim, **kw)
        # gates start near 1: a state that lasts some tens of frames
        nn.init.constant_(self.inner.bias[dim:].detach(), 2.0)

    def _map(self, x):
        return self.down(self.up(self.norm2(x)), x)

    def forward(self, x, state=None, lengths=None):
        value, gate = self.inner(self.norm1(x)).split(x.shape[-1], -1)
        h, state = gated_scan(value, gate, state, lengths=lengths)
        return self._map(self.outer(h, x)), state

    @torch.no_grad()
    def step(self, x, state):
        value, gate = self.inner(self.norm1(x)).split(x.shape[-1], -1)
        return self._map(self.outer(gated_scan_step(value, gate, state), x))


class SequenceEncoder(nn.Module):
    """Frames [B,T,in_features] to features [B,T,dim] for an alignment loss.

    ``forward(x, lengths=None)`` encodes whole sequences.  ``init_state(batch)`` and
    ``step(x_t, states)`` encode a live stream frame by frame, with the same result.
    """

    def __init__(self, in_features, dim, layers=2, hidden=None, *, device=None, dtype=None):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        self.dim = int(dim)
        self.embed = Linear(in_features, dim, **kw)
        self.blocks = nn.ModuleList(EncoderBlock(dim, hidden, **kw) for _ in range(layers))
        self.norm = LayerNorm(dim, **kw)

    def forward(self, x, lengths=None):
        x = self.embed(x)
        for block in self.blocks:
            x, _ = block(x, None, lengths)
        return self.norm(x)

    def init_state(self, batch):
        """The states before the first frame, one float32 [batch, dim] tensor a block."""
        kw = {"dtype": torch.float32, "device": self.embed.weight.device}
        return [torch.zeros(batch, self.dim, **kw) for _ in self.blocks]

    @torch.no_grad()
    def step(self, x, states):
        """One frame [B,in_features]; ``states`` are updated in place."""
        x = self.embed(x)
        for block, state in zip(self.blocks, states):
            x = block.step(x, state)
        return self.norm(x)
