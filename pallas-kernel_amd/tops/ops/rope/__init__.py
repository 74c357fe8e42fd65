"""Norms of queries and keys for each head with the rotary position embedding in the same pass.
The reference has no such operator."""

from .qk_norm_rope import qk_norm_rope, rotary_inv_freq

__all__ = ["qk_norm_rope", "rotary_inv_freq"]
