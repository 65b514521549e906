"""Policy operators: from a network's features to the action, and its training.

The environment hands out observations and legal masks and takes actions;
these are the hand-written CUDA operators in between (``jq_layer_norm``,
``jq_action_log_prob``, ``jq_verify_drafts`` of ``include/jq.h``):

* :func:`layer_norm` -- forward and backward;
* :func:`action_log_prob` -- log-probability of an action and entropy over
  the legal set, with their gradient: what PPO's loss is made of;
* :func:`sample_actions` -- one action per row from given random numbers;
* :func:`verify_drafts` -- keeps of some drafted plies what is distributed as
  the target policy's own play, and draws the ply behind them;
* :class:`PolicyHead` -- the module made of them, whose :meth:`~PolicyHead.policy`
  is a policy for :class:`junqi_b200.collector.RolloutCollector`.

Logits and features are float32, float16 or bfloat16; masks are the
environment's own (uint8 or bool, nonzero: legal), or None.  Masks and actions
are read during the call: those of the environment, the history and the
collector are buffers that their next call overwrites, so the backward pass
keeps its own copy, the mask's in bits.
Everything runs on the current stream of the tensors' device, synchronises
nothing, and may be captured into a CUDA graph.  A backward pass that is
captured needs leaves that no earlier eager graph still refers to: release
eager losses and outputs before the capture, as for any torch module.

Nothing here falls back to torch: wrong arguments raise ValueError, a failed
call RuntimeError.  Inputs with a forward-mode tangent are refused.
"""
from __future__ import annotations

from typing import Callable, NamedTuple

import torch

from . import _native as N

NUM_ACTIONS = 129 * 129  # compact canonical actions cs * 129 + cd


class Verified(NamedTuple):
    accepted: torch.Tensor   # (games,) int32: drafted actions kept
    actions: torch.Tensor    # (games, drafts + 1) int32: those, the drawn action, then -1
    log_probs: torch.Tensor  # (games, drafts + 1) float32: the target's, 0 behind them


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of ``x`` (..., dim).

    ``weight`` and ``bias`` are (dim,), float32 or of x's type (both alike), or
    None.  Statistics are 32-bit; the result has x's type.  Differentiable once
    with respect to x, weight and bias."""
    return N.policy().layer_norm(x, weight, bias, eps)


def action_log_prob(logits: torch.Tensor, mask: torch.Tensor | None,
                    actions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(log-probability of ``actions`` (...), entropy (...)) of the softmax of
    ``logits`` (..., n) over each row's legal places, float32.

    ``mask`` is uint8 or bool, (..., n) or broadcast to it; None: all legal.
    What stands at masked places is never looked at.  An action outside
    [0, n) (the samplers' -1 included) is "no action": log-probability 0 and no
    gradient.  One that is not legal has log-probability -inf and no gradient.
    A row without legal places has entropy 0.  NaN or +inf at a legal place
    gives NaN.  Differentiable once with respect to ``logits``."""
    return N.policy().action_log_prob(logits, mask, actions)


def verify_drafts(logits: torch.Tensor, drafts: torch.Tensor, accept_u: torch.Tensor, sample_u: torch.Tensor, *,
                  draft_logits: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                  lengths: torch.Tensor | None = None) -> Verified:
    """Verify D drafted actions per game against the target policy.

    ``logits`` (games, D + 1, n): the target's at each drafted place and at the
    one behind the last; ``drafts`` (games, D) the drafted actions;
    ``draft_logits`` (games, D, n), of the same type: those they were drawn
    from, or None where the draft is certain of its action; ``mask`` uint8 or
    bool, (games, D + 1, n) or broadcast to it, the legal set of both; ``lengths``
    (games,) how many drafts each game uses (None: all).  ``accept_u`` (games, D)
    and ``sample_u`` (games,) are random numbers in [0, 1), float32.

    A drafted action is kept while accept_u q(a) < p(a); at the first that is
    not, the action is drawn from max(p - q, 0), after the last from p.  The
    actions that come out are distributed as if the target had played alone.
    The choices are those of 64-bit arithmetic, with exponentials that are good to
    2^-42 and 0 below e^-700; log-probabilities are rounded from it once (those of
    kept drafts without a mask come from 32-bit sums: off by (92 + 6 n / 256) 2^-24
    at most, measured below 2^-17 up to 262,144 actions).  A place without legal
    actions gives -1, one with NaN or +inf at a legal place -1 and a NaN
    log-probability.  Not differentiable: see :func:`action_log_prob`.

    An environment does not go back to the ply of a rejection: draft on a batch of
    which another one holds the positions to play on from."""
    return Verified(*N.policy().verify_drafts(logits, drafts, accept_u, sample_u, draft_logits, mask, lengths))


def sample_actions(logits: torch.Tensor, mask: torch.Tensor | None,
                   u: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(actions (...) int32, their log-probabilities (...) float32), one per row of
    ``logits`` (..., n), drawn from the softmax over the legal places: the least
    action whose running probability exceeds ``u`` (...), random numbers in [0, 1).
    A row without legal actions gives -1 (``jq_ply`` takes it as no move)."""
    return N.policy().sample_actions(logits, mask, u)


# -- the head -----------------------------------------------------------------------------

class PolicyHead(torch.nn.Module):
    """A trunk's features (..., features) to logits over the canonical actions and a
    value: layer norm, then one linear map each.

    ``policy(trunk)`` is a policy for ``RolloutCollector``, where
    ``trunk(spatial, global) -> features``; on a minibatch that
    ``RolloutHistory.reconstruct`` rebuilt, ``evaluate`` gives what the loss
    needs; ``verify`` checks plies that a cheaper policy drafted."""

    def __init__(self, features: int, actions: int = NUM_ACTIONS, eps: float = 1e-5, device=None, dtype=None):
        super().__init__()
        self.eps = float(eps)
        self.weight = torch.nn.Parameter(torch.ones(features, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(features, device=device, dtype=dtype))
        self.action = torch.nn.Linear(features, actions, device=device, dtype=dtype)
        self.value = torch.nn.Linear(features, 1, device=device, dtype=dtype)

    def forward(self, features: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        h = layer_norm(features, self.weight, self.bias, self.eps)
        return self.action(h), self.value(h).squeeze(-1).float()

    def policy(self, trunk: Callable[[torch.Tensor, torch.Tensor], torch.Tensor]):
        """policy(spatial, global, mask) -> (logits, value): the collector draws the actions."""
        return lambda spatial, global_, mask: self(trunk(spatial, global_))

    def evaluate(self, features: torch.Tensor, mask: torch.Tensor | None, actions: torch.Tensor):
        """(log-probabilities, entropies, values) of ``actions``, with gradients."""
        logits, value = self(features)
        lp, ent = action_log_prob(logits, mask, actions)
        return lp, ent, value

    def verify(self, features: torch.Tensor, drafts: torch.Tensor, accept_u: torch.Tensor, sample_u: torch.Tensor,
               **kw) -> Verified:
        """:func:`verify_drafts` of plies whose features are (games, drafts + 1, features)."""
        with torch.no_grad():
            return verify_drafts(self(features)[0], drafts, accept_u, sample_u, **kw)
