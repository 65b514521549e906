"""Refusals of the policy operators that need no GPU, at the ends of what they take."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from junqi_b200 import policy as P


@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "logits"])
def test_forward_mode_is_refused(which, needs_grad):
    """A tangent is an error, never dropped; without one, or where tangents are switched off, the next check speaks."""
    args = {k: torch.ones(s) for k, s in (("x", (2, 3, 4)), ("weight", (4,)), ("bias", (4,)), ("logits", (3, 4)))}

    def call():
        if which == "logits":
            return P.action_log_prob(args["logits"], None, torch.zeros(3, dtype=torch.int32))
        return P.layer_norm(args["x"], args["weight"], args["bias"])

    with pytest.raises(ValueError, match="CUDA"):
        call()
    primal, tangent = args[which].requires_grad_(needs_grad), torch.ones_like(args[which])
    with fwd.dual_level():
        args[which] = fwd.make_dual(primal, tangent)
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="no forward-mode derivative"):
            call()
        with fwd._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="CUDA"):
        call()
