"""Layer norm over the last dimension. The reference has the root-mean-square norm alone."""

from .layer_norm import layer_norm

__all__ = ["layer_norm"]
