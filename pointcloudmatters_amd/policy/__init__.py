"""Policies and point-cloud tokenizers of the BC path (reference: src/models/components/)."""
from .act import ACTPCD, ACTRLBenchPCD
from .cross_attn import cross_attention
from .gated import gated_ffn
from .losses import KLDivergence
from .pointnet import PointNet
from .rotary import rotary_axes
from .transformer import Transformer, TransformerEncoder

__all__ = ["ACTPCD", "KLDivergence", "PointNet", "Transformer", "TransformerEncoder", "cross_attention", "gated_ffn", "rotary_axes"]
