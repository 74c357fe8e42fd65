"""The forms that update a state in place have no tangents either: inputs that carry one are refused,
also under no_grad, which leaves forward-mode differentiation on."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_delta_refusals import step_args
from tops.ops.delta import gated_delta_rule_step


@pytest.mark.parametrize("name", ["state", "q", "k", "v", "g", "beta"])
def test_step(name):
    a = step_args()
    with torch.no_grad(), fwd.dual_level():
        a[name] = fwd.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(RuntimeError, match="tangent"):
            gated_delta_rule_step(**a)


def test_nothing_to_differentiate():
    """It goes on to the next check."""
    with torch.no_grad(), fwd.dual_level():
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            gated_delta_rule_step(**step_args())
