"""The gated delta rule: a linear attention whose state gives up what a key held before the key
writes anew. For prompts and training, and for the next tokens of a serving batch. The reference
has no such operator."""

from .gated_delta_rule import gated_delta_rule, gated_delta_rule_step

__all__ = ["gated_delta_rule", "gated_delta_rule_step"]
