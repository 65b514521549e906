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
environment's own (uint8 or bool, nonzero: legal), or None.  A mask is read
during the call: the environment's and the history's masks are buffers that
their next call overwrites, so the backward pass keeps its own copy, in bits.
Everything runs on the current stream of the tensors' device, synchronises
nothing, and may be captured into a CUDA graph.  A backward pass that is
captured needs leaves that no earlier eager graph still refers to: release
eager losses and outputs before the capture, as for any torch module.

Nothing here falls back to torch: wrong arguments raise ValueError, a failed
call RuntimeError.
"""
from __future__ import annotations

import ctypes
from typing import Callable, NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

NUM_ACTIONS = 129 * 129  # compact canonical actions cs * 129 + cd

_DTYPES = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}
_INTS = (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64)


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream(i).cuda_stream, without 10 us of wrapping


def _call(name: str, device: torch.device, *args) -> None:
    """Entry point ``name`` on the current stream of ``device``, made current for the call."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _call(name, device, *args)
    status = getattr(N.lib(), name)(*args, _raw_stream(device.index))
    if status:
        N.check(status, name)


def _device(what: str, *tensors: torch.Tensor | None) -> torch.device:
    """The one CUDA device of all tensors."""
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    if dev.type != "cuda":
        raise ValueError(f"{what}: needs CUDA tensors, got {dev}")
    return dev


def _last(t: torch.Tensor) -> torch.Tensor:
    """`t` with neighbouring places next to each other on its last axis."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(rows, n) view of `t` (a copy only where its leading axes have no common stride)."""
    return _last(t if t.dim() == 2 else t.reshape(-1, t.shape[-1]))


def _float_dtype(what: str, t: torch.Tensor) -> int:
    if t.dtype not in _DTYPES:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return _DTYPES[t.dtype]


def _int32(what: str, t: torch.Tensor, shape, lo: int, hi: int) -> torch.Tensor:
    """`t` as contiguous int32 of `shape`; 64-bit values are cut to [lo, hi] first, so that none wraps."""
    if t.dtype not in _INTS:
        raise ValueError(f"{what} must be whole numbers, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype == torch.int64:
        t = t.clamp(lo, hi)
    return t.to(torch.int32).contiguous()


def _mask_for(what: str, mask: torch.Tensor | None, shape) -> torch.Tensor | None:
    """`mask` as uint8, expanded to `shape`."""
    if mask is None:
        return None
    if mask.dtype not in (torch.uint8, torch.bool):
        raise ValueError(f"{what}: the mask must be uint8 or bool, got {mask.dtype}")
    try:
        mask = mask.expand(shape)
    except RuntimeError:
        raise ValueError(f"{what}: a mask of {tuple(mask.shape)} does not fit logits of {tuple(shape)}") from None
    return mask.view(torch.uint8)


def _wants_grad(*tensors: torch.Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# -- layer norm -----------------------------------------------------------------

def _norm_forward(shape, x2, weight, bias, eps, stats):
    rows, dim = x2.shape
    y = torch.empty(shape, dtype=x2.dtype, device=x2.device)
    if rows:
        w = weight if weight is not None else bias
        _call("jq_layer_norm", x2.device, x2.data_ptr(), x2.stride(0), _ptr(weight), _ptr(bias), rows, dim,
              _DTYPES[x2.dtype], N.F32 if w is None else _DTYPES[w.dtype], eps, y.data_ptr(), _ptr(stats))
    return y


def _norm_scratch(device, rows, dim):
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _norm_scratch(device, rows, dim)
    return N.lib().jq_layer_norm_scratch_floats(rows, dim)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = _rows(x)
        stats = torch.empty((x2.shape[0], 3), dtype=torch.float32, device=x.device)
        ctx.save_for_backward(x2, weight, bias, stats)
        return _norm_forward(x.shape, x2, weight, bias, eps, stats)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, weight, bias, stats = ctx.saved_tensors
        rows, dim = x2.shape
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty(dy.shape, dtype=x2.dtype, device=x2.device) if need_x else None
        dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if need_w else None
        db = torch.empty_like(bias, memory_format=torch.contiguous_format) if need_b else None
        if rows:
            dy2 = _rows(dy)
            w = weight if weight is not None else bias
            part = torch.empty(_norm_scratch(x2.device, rows, dim), dtype=torch.float32,
                               device=x2.device) if need_w or need_b else None
            _call("jq_layer_norm_backward", x2.device, x2.data_ptr(), x2.stride(0), _ptr(weight), dy2.data_ptr(),
                  dy2.stride(0), stats.data_ptr(), rows, dim, _DTYPES[x2.dtype],
                  N.F32 if w is None else _DTYPES[w.dtype], _ptr(dx), _ptr(dw), _ptr(db), _ptr(part))
        else:
            for g in (dw, db):
                if g is not None:
                    g.zero_()
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of ``x`` (..., dim).

    ``weight`` and ``bias`` are (dim,), float32 or of x's type (both alike), or
    None.  Statistics are 32-bit; the result has x's type.  Differentiable once
    with respect to x, weight and bias."""
    _float_dtype("layer_norm: x", x)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: x needs a last axis, got {tuple(x.shape)}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if tuple(p.shape) != (x.shape[-1],):
            raise ValueError(f"layer_norm: {name} must be ({x.shape[-1]},), got {tuple(p.shape)}")
        if p.dtype not in (torch.float32, x.dtype):
            raise ValueError(f"layer_norm: {name} must be float32 or {x.dtype}, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("layer_norm: weight and bias must have one type")
    _device("layer_norm", x, weight, bias)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm_forward(x.shape, _rows(x), weight, bias, float(eps), None)


# -- log-probability and entropy ----------------------------------------------------

def _logp_forward(shape, x2, m2, act, stats, bits):
    rows, n = x2.shape
    lp, ent = (torch.empty(shape, dtype=torch.float32, device=x2.device) for _ in range(2))
    if rows:
        _call("jq_action_log_prob", x2.device, x2.data_ptr(), x2.stride(0), _DTYPES[x2.dtype], _ptr(m2),
              0 if m2 is None else m2.stride(0), act.data_ptr(), rows, n, lp.data_ptr(), ent.data_ptr(), _ptr(stats),
              _ptr(bits))
    return lp, ent


class _ActionLogProb(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, act):
        x2 = _rows(logits)
        m2 = None if mask is None else _rows(mask)
        rows, n = x2.shape
        stats = torch.empty((rows, 4), dtype=torch.float32, device=x2.device)
        bits = None if mask is None else torch.empty((rows, (n + 31) // 32), dtype=torch.int32, device=x2.device)
        ctx.save_for_backward(x2, act, stats, bits)
        ctx.shape = logits.shape
        ctx.set_materialize_grads(False)
        return _logp_forward(logits.shape[:-1], x2, m2, act, stats, bits)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent):
        if g_lp is None and g_ent is None:
            return None, None, None
        x2, act, stats, bits = ctx.saved_tensors
        rows, n = x2.shape
        dx = torch.empty(ctx.shape, dtype=x2.dtype, device=x2.device)
        if rows:
            g_lp, g_ent = (None if g is None else g.reshape(-1) for g in (g_lp, g_ent))
            _call("jq_action_log_prob_backward", x2.device, x2.data_ptr(), x2.stride(0), _DTYPES[x2.dtype],
                  _ptr(bits), act.data_ptr(), stats.data_ptr(), _ptr(g_lp), 0 if g_lp is None else g_lp.stride(0),
                  _ptr(g_ent), 0 if g_ent is None else g_ent.stride(0), rows, n, dx.data_ptr())
        return dx, None, None


def _check_actions(what: str, logits: torch.Tensor, dim: int | None = None) -> int:
    _float_dtype(f"{what}: logits", logits)
    if logits.dim() < 1 or (dim is not None and logits.dim() != dim):
        raise ValueError(f"{what}: logits of {tuple(logits.shape)}")
    n = logits.shape[-1]
    if not 0 < n <= N.POLICY_MAX_ACTIONS:
        raise ValueError(f"{what}: 1 to {N.POLICY_MAX_ACTIONS} actions, got {n}")
    return n


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
    n = _check_actions("action_log_prob", logits)
    act = _int32("action_log_prob: actions", actions, logits.shape[:-1], -1, n).view(-1)
    mask = _mask_for("action_log_prob", mask, logits.shape)
    _device("action_log_prob", logits, mask, act)
    if _wants_grad(logits):
        return _ActionLogProb.apply(logits, mask, act)
    return _logp_forward(logits.shape[:-1], _rows(logits), None if mask is None else _rows(mask), act, None, None)


# -- sampling and verification ----------------------------------------------------------

class Verified(NamedTuple):
    accepted: torch.Tensor   # (games,) int32: drafted actions kept
    actions: torch.Tensor    # (games, drafts + 1) int32: those, the drawn action, then -1
    log_probs: torch.Tensor  # (games, drafts + 1) float32: the target's, 0 behind them


def _uniform(what: str, u: torch.Tensor, shape) -> torch.Tensor:
    if u.dtype != torch.float32 or tuple(u.shape) != tuple(shape):
        raise ValueError(f"{what} must be float32 {tuple(shape)}, got {u.dtype} {tuple(u.shape)}")
    return u.contiguous()


def _verify(x, drafts, accept_u, sample_u, y, mask, lengths):
    games, places, n = x.shape
    acc, out = (torch.empty(s, dtype=torch.int32, device=x.device) for s in ((games,), (games, places)))
    lp = torch.empty((games, places), dtype=torch.float32, device=x.device)
    if games:
        d = N.JqDrafts(games=games, drafts=places - 1, actions=n, dtype=_DTYPES[x.dtype], logits=x.data_ptr(),
                       logits_game=x.stride(0), logits_place=x.stride(1), drafted=_ptr(drafts), lengths=_ptr(lengths),
                       accept_u=_ptr(accept_u), sample_u=sample_u.data_ptr(), accepted=acc.data_ptr(),
                       out_actions=out.data_ptr(), log_probs=lp.data_ptr())
        if y is not None:
            d.draft_logits, d.draft_game, d.draft_place = y.data_ptr(), y.stride(0), y.stride(1)
        if mask is not None:
            d.mask, d.mask_game, d.mask_place = mask.data_ptr(), mask.stride(0), mask.stride(1)
        _call("jq_verify_drafts", x.device, ctypes.byref(d))
    return Verified(acc, out, lp)


@torch.no_grad()
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
    Computed in 64 bits; ties go to the lowest action.  A place without legal
    actions gives -1, one with NaN or +inf at a legal place -1 and a NaN
    log-probability.  Not differentiable: see :func:`action_log_prob`."""
    n = _check_actions("verify_drafts", logits, 3)
    games, places = logits.shape[:2]
    if not 1 <= places <= N.POLICY_MAX_DRAFTS + 1:
        raise ValueError(f"verify_drafts: 1 to {N.POLICY_MAX_DRAFTS + 1} places a game, got {places}")
    drafts = _int32("verify_drafts: drafts", drafts, (games, places - 1), -1, n)
    accept_u = _uniform("verify_drafts: accept_u", accept_u, (games, places - 1))
    sample_u = _uniform("verify_drafts: sample_u", sample_u, (games,))
    if draft_logits is not None:
        if draft_logits.dtype != logits.dtype or tuple(draft_logits.shape) != (games, places - 1, n):
            raise ValueError(f"verify_drafts: draft_logits must be {logits.dtype} {(games, places - 1, n)}, got "
                             f"{draft_logits.dtype} {tuple(draft_logits.shape)}")
        draft_logits = _last(draft_logits)
    if lengths is not None:
        lengths = _int32("verify_drafts: lengths", lengths, (games,), 0, places - 1)
    mask = _mask_for("verify_drafts", mask, logits.shape)
    _device("verify_drafts", logits, drafts, accept_u, sample_u, draft_logits, mask, lengths)
    return _verify(_last(logits), drafts, accept_u, sample_u, draft_logits, None if mask is None else _last(mask),
                   lengths)


@torch.no_grad()
def sample_actions(logits: torch.Tensor, mask: torch.Tensor | None,
                   u: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(actions (...) int32, their log-probabilities (...) float32), one per row of
    ``logits`` (..., n), drawn from the softmax over the legal places: the least
    action whose running probability exceeds ``u`` (...), random numbers in [0, 1).
    A row without legal actions gives -1 (``jq_ply`` takes it as no move)."""
    _check_actions("sample_actions", logits)
    shape = logits.shape[:-1]
    u = _uniform("sample_actions: u", u, shape)
    mask = _mask_for("sample_actions", mask, logits.shape)
    _device("sample_actions", logits, mask, u)
    v = _verify(_rows(logits)[:, None], None, None, u.view(-1), None, None if mask is None else _rows(mask)[:, None],
                None)
    return v.actions.view(shape), v.log_probs.view(shape)


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
