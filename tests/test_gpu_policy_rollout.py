"""The policy operators as they are used together: a head plays a rollout through the collector, the history gives
the minibatch back, the loss is trained on it, and drafted plies are verified."""
from __future__ import annotations

import pytest
import torch

from junqi_b200 import _native as N
from junqi_b200 import policy as P
from junqi_b200 import tables
from junqi_b200.collector import RolloutCollector
from junqi_b200.env import HALF_DARK, JunqiEnvB200

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def trunk(sp, gl):
    """A stand-in: what stands on each row of the board, with the globals (40 channels of 17 rows, 28)."""
    return torch.cat([sp[:, :40].sum(3).flatten(1), gl], 1)


def _env(n, seed):
    env = JunqiEnvB200(n, show_mode=HALF_DARK, pool=tables.build_setup_pool(48, seed=2), rules=N.RULES_GAMESTATE)
    env.reset(seed=seed)
    return env


def _head(seed=0):
    torch.manual_seed(seed)
    head = P.PolicyHead(40 * 17 + 28, device="cuda")
    with torch.no_grad():
        head.action.weight.mul_(8)
    return head


@pytest.mark.parametrize("graph", [False, True])
def test_head_plays_trains_and_is_scored_alike(graph):
    n, T = 64, 12
    env, head = _env(n, 3), _head()
    col = RolloutCollector(env, head.policy(trunk), T, seed=1, graph=graph)
    torch.manual_seed(5)
    r = col.collect()
    first = r.actions.clone()
    assert int(env.stats[5]) == n * T, "an action was not legal"
    # the minibatch as training sees it: same positions, same masks, same scores
    idx = torch.randperm(n * T, device="cuda")[:96]
    mb = r.history.reconstruct(idx)
    acts, old = r.actions.view(-1)[idx], r.log_probs.view(-1)[idx]
    lp, ent, value = head.evaluate(trunk(mb["spatial"], mb["global"]), mb["mask"], acts)
    # the same formula on logits that a product of another batch size left: 708 terms of 32 bits of about 8
    assert (lp - old).abs().max() < 708 * U * 8 * 8
    assert ((value - r.values.view(-1)[idx]).abs() < 708 * U * 8 * 8).all()
    assert (lp < 0).any() and torch.isfinite(lp).all() and (ent > 0).any()
    loss = -(torch.exp(lp - old) * torch.linspace(-1, 1, 96, device="cuda")).mean() - 0.01 * ent.mean() + value.square().mean()
    r.history.reconstruct(idx.flip(0))  # overwrites the mask buffer between forward and backward
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in head.parameters())
    assert head.weight.grad.any() and head.action.weight.grad.any()
    assert not torch.equal(col.collect().actions, first)


def test_head_gradients_against_plain_modules():
    """The whole head in 64 bits by torch's own modules."""
    env, head = _env(32, 8), _head(2)
    sp, gl = env.observe()
    mask = env.mask.clone()
    feats = trunk(sp, gl).detach()
    acts, _ = P.sample_actions(head(feats)[0], mask, torch.rand(32, device="cuda"))
    lp, ent, value = head.evaluate(feats, mask, acts)
    (lp.mean() + 0.1 * ent.mean() + value.mean()).backward()
    import copy
    ref = copy.deepcopy(head).double()
    for p in ref.parameters():
        p.grad = None
    h = torch.nn.functional.layer_norm(feats.double(), (feats.shape[1],), ref.weight, ref.bias, head.eps)
    logp = torch.log_softmax(ref.action(h).masked_fill(mask == 0, -torch.inf), 1)
    e = -(logp.exp() * torch.where(mask != 0, logp, 0)).sum(1)  # a gradient without 0 * inf at masked places
    (logp.gather(1, acts.long()[:, None]).mean() + 0.1 * e.mean() + ref.value(h).mean()).backward()
    for (name, p), q in zip(head.named_parameters(), ref.parameters()):
        # logits of 708 products of 32 bits (TF32 is off by default) move the gradient by about 708 u relative
        err = (p.grad.double() - q.grad).norm() / q.grad.norm()
        assert err < 4 * 708 * U, (name, float(err))


def test_drafted_plies_are_verified():
    """A cheap head plays D plies; the large one scores the recorded positions at once and keeps what is its own."""
    n, D = 48, 4
    env, cheap, large = _env(n, 11), _head(1), _head(1)
    with torch.no_grad():
        large.action.weight.add_(0.05 * torch.randn_like(large.action.weight))
    from junqi_b200.history import RolloutHistory
    hist = RolloutHistory(D + 1, n)
    drafts, q = [], []
    for t in range(D + 1):
        hist.snapshot(env.batch, t)
        if t == D:
            break
        sp, gl = env.observe()
        with torch.no_grad():
            logits, _ = cheap(trunk(sp, gl))
        a, _ = P.sample_actions(logits, env.mask, torch.rand(n, device="cuda"))
        drafts.append(a)
        q.append(logits)
        world = torch.empty(n, dtype=torch.int32, device="cuda")
        import ctypes
        N.check(N.lib().jq_canonical_to_world(ctypes.byref(env.batch.struct), a.data_ptr(), None, world.data_ptr(),
                                              torch.cuda.current_stream().cuda_stream), "jq_canonical_to_world")
        env.ply(world, seed=1, ply=t + 1, autoreset=False)
    at = (torch.arange(n)[:, None] + n * torch.arange(D + 1)[None, :]).flatten()
    mb = hist.reconstruct(at)
    feats = trunk(mb["spatial"], mb["global"]).view(n, D + 1, -1)
    mask = mb["mask"].view(n, D + 1, -1)
    drafts, q = torch.stack(drafts, 1), torch.stack(q, 1)
    au, su = torch.rand(n, D, device="cuda"), torch.rand(n, device="cuda")
    v = large.verify(feats, drafts, au, su, draft_logits=q, mask=mask)
    step = torch.arange(D + 1, device="cuda")[None, :]
    kept = step < v.accepted[:, None]
    assert torch.equal(v.actions[:, :D][kept[:, :D]], drafts[kept[:, :D]])
    assert (v.actions[step > v.accepted[:, None]] == -1).all()
    assert 0 < int(v.accepted.sum()) < n * D
    real = v.actions >= 0
    assert mask.gather(2, v.actions.clamp(min=0).long()[..., None])[..., 0][real].all(), "an illegal action"
    with torch.no_grad():
        lp, _ = P.action_log_prob(large(feats)[0], mask, v.actions)
    # the same logits, scored in 32 and in 64 bits: (16641 / 256 + 28 + 60) u, and rounding
    assert ((lp - v.log_probs)[real].abs() < 400 * U).all()
    # the large head on its own drafts keeps them all
    same = cheap.verify(feats, drafts, au, su, draft_logits=cheap(feats[:, :D])[0], mask=mask)
    assert (same.accepted >= v.accepted).float().mean() > 0.9
