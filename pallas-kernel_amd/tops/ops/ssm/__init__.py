"""Selective state space operators: the scan and its short causal convolution, for prompts and
training, and their single-token forms for serving. The reference has none of them."""

from .conv import causal_conv1d, causal_conv1d_step
from .scan import selective_scan, selective_scan_step

__all__ = ["causal_conv1d", "causal_conv1d_step", "selective_scan", "selective_scan_step"]
