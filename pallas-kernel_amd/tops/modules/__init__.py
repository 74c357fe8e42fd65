"""Layer building blocks on the MI355X kernels (mirror of the reference's ``tops.modules``, and
``LayerNorm`` beside them)."""

from .convolution import ShortConvolution
from .fused_norm_gate import FusedRMSNormGated
from .layernorm import LayerNorm, RMSNorm

__all__ = ["FusedRMSNormGated", "LayerNorm", "RMSNorm", "ShortConvolution"]
