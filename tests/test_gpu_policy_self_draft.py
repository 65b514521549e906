"""A policy that verifies its own drafts keeps them all."""
from __future__ import annotations

import ctypes

import pytest
import torch

from junqi_b200 import _native as N
from junqi_b200 import policy as P
from junqi_b200.history import RolloutHistory
from tests.test_gpu_policy_rollout import _env, _head, trunk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_own_drafts_are_all_kept(dtype, masked):
    """Plies that a head played, scored once: target and draft have the same logits, so p = q bit by bit and u q < p for
    every u below 1 (the largest is 1 - 2^-24, far from 1 in 64 bits)."""
    n, D = 48, 5
    env, head = _env(n, 17), _head(4)
    hist = RolloutHistory(D + 1, n)
    for t in range(D + 1):
        hist.snapshot(env.batch, t)
        if t == D:
            break
        with torch.no_grad():
            logits, _ = head(trunk(*env.observe()))
        a, _ = P.sample_actions(logits, env.mask, torch.rand(n, device="cuda"))
        world = torch.empty(n, dtype=torch.int32, device="cuda")
        N.check(N.lib().jq_canonical_to_world(ctypes.byref(env.batch.struct), a.data_ptr(), None, world.data_ptr(),
                                              torch.cuda.current_stream().cuda_stream), "jq_canonical_to_world")
        env.ply(world, seed=1, ply=t + 1, autoreset=False)
    mb = hist.reconstruct((torch.arange(n)[:, None] + n * torch.arange(D + 1)[None, :]).flatten())
    mask = mb["mask"].view(n, D + 1, -1) if masked else None
    with torch.no_grad():
        logits = head(trunk(mb["spatial"], mb["global"]))[0].view(n, D + 1, -1).to(dtype)
    drafts, lp = P.sample_actions(logits[:, :D], None if mask is None else mask[:, :D], torch.rand(n, D, device="cuda"))
    some = torch.ones(n, D, dtype=torch.bool, device="cuda") if mask is None else mask[:, :D].bool().any(-1)
    assert torch.equal(drafts >= 0, some) and some.all(1).sum() > n // 2
    want = some.long().cumprod(1).sum(1)  # a finished game ends there
    for u in (torch.rand(n, D, device="cuda"), torch.full((n, D), 1 - 2.0 ** -24, device="cuda"), torch.zeros(n, D, device="cuda")):
        v = P.verify_drafts(logits, drafts, u, torch.rand(n, device="cuda"), draft_logits=logits[:, :D].clone(), mask=mask)
        assert torch.equal(v.accepted.long(), want)
        kept = torch.arange(D, device="cuda")[None, :] < want[:, None]
        assert torch.equal(v.actions[:, :D][kept], drafts[kept])
        # rounded once from 64 bits twice, or (without a mask) once from a 32-bit sum: (92 + 6 * 16641 / 256) u
        tol = (2 * lp.abs() + (0 if masked else 92 + 6 * 66)) * 2.0 ** -24 + 2.0 ** -40
        assert ((v.log_probs[:, :D] - lp).abs() <= tol)[kept].all()
