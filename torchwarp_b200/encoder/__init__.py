"""Sequence encoders in front of an alignment loss: layer norm, linear with its epilogue, the
gated linear recurrence, the modules made of them, and AdamW."""

from .functional import GatedScanOutput, gated_scan, gated_scan_step, layer_norm, linear
from .module import EncoderBlock, LayerNorm, Linear, SequenceEncoder
from .optim import AdamW

__all__ = ["GatedScanOutput", "gated_scan", "gated_scan_step", "layer_norm", "linear",
           "EncoderBlock", "LayerNorm", "Linear", "SequenceEncoder", "AdamW"]
