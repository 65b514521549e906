"""The policy operators' refusals that need no GPU, at the ends of what they take, and the build of their binding."""
from __future__ import annotations

import importlib.metadata
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwd

from junqi_b200 import _native as N
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


def test_the_binding_is_built_for_this_interpreter_and_torch(tmp_path, monkeypatch):
    """`make` gets the running interpreter; a binding of another Python or torch is refused, and built anew."""
    assert N._policy_is_ours()
    assert N.policy().built_for.endswith(f"{sys.implementation.cache_tag} torch-{importlib.metadata.version('torch')}")
    other = tmp_path / "_policy.so"
    other.write_bytes(N.POLICY_PATH.read_bytes().replace(importlib.metadata.version("torch").encode() + b"\0", b"0.0\0"))
    calls = []
    monkeypatch.setattr(N, "POLICY_PATH", other)
    monkeypatch.setattr(N, "_policy", None)
    monkeypatch.setattr(N.subprocess, "run", lambda cmd, check: calls.append(cmd))
    with pytest.raises(RuntimeError, match="another Python or torch"):
        N.policy()
    N.build()
    assert not other.exists() and f"PYTHON={sys.executable}" in calls[0]


@pytest.mark.parametrize("kind", [tuple, list, iter, lambda out: (v for v in out), torch.stack])
def test_the_collector_takes_what_can_be_unpacked(kind):
    """(action, log_prob, value) in whatever form a policy returns it: an iterator has no length, and no last element."""
    from types import SimpleNamespace

    from junqi_b200.collector import RolloutCollector
    mask, want = torch.ones(2, 4, dtype=torch.uint8), [torch.full((2,), float(k)) for k in (1, 2, 3)]
    col = RolloutCollector.__new__(RolloutCollector)
    col.env = SimpleNamespace(observe=lambda seats, seats_per_env: (None, None), mask=mask, n=2, device="cpu",
                              batch={"terminated": torch.tensor([0, 1])})
    col.policy = lambda sp, gl, m: kind(want)
    col.last_values = torch.zeros(2)
    for got, w in zip(col._act(), want):
        assert torch.equal(got, w)
    col._final()
    assert col.last_values.tolist() == [3.0, 0.0]
