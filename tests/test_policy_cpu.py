"""Refusals of the policy operators, and their binding, without a GPU."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from junqi_b200 import _native as N
from junqi_b200 import policy as P

ROOT = Path(__file__).resolve().parent.parent
F, H, I = torch.float32, torch.float16, torch.int32


def t(*shape, dtype=F):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("args,text", [
    ((t(3, 4, dtype=torch.float64),), "float32, float16 or bfloat16"),
    ((t(3, 0),), "last axis"),
    ((t(),), "last axis"),
    ((t(3, 4), t(5)), "weight must be"),
    ((t(3, 4), t(4), t(1, 4)), "bias must be"),
    ((t(3, 4, dtype=H), t(4, dtype=torch.bfloat16)), "weight must be float32 or"),
    ((t(3, 4, dtype=H), t(4), t(4, dtype=H)), "one type"),
    ((t(3, 4), None, None, -1e-5), "eps"),
    ((t(3, 4), None, None, float("nan")), "eps"),
    ((t(3, 4), t(4), t(4)), "CUDA"),
])
def test_layer_norm_refuses(args, text):
    with pytest.raises(ValueError, match=text):
        P.layer_norm(*args)


@pytest.mark.parametrize("args,text", [
    ((t(3, 4, dtype=torch.float64), None, t(3, dtype=I)), "float32, float16 or bfloat16"),
    ((t(3, 0), None, t(3, dtype=I)), "actions"),
    ((t(), None, t(dtype=I)), "logits"),
    ((t(1, N.POLICY_MAX_ACTIONS + 1), None, t(1, dtype=I)), "actions"),
    ((t(3, 4), None, t(3)), "whole numbers"),
    ((t(3, 4), None, t(3, dtype=torch.bool)), "whole numbers"),
    ((t(3, 4), None, t(4, dtype=I)), r"actions must be \(3,\)"),
    ((t(3, 4), None, t(3, 1, dtype=I)), r"actions must be \(3,\)"),
    ((t(3, 4), t(3, 4), t(3, dtype=I)), "mask must be uint8 or bool"),
    ((t(3, 4), t(3, 5, dtype=torch.bool), t(3, dtype=I)), "does not fit"),
    ((t(3, 4), t(2, 3, 4, dtype=torch.bool), t(3, dtype=I)), "does not fit"),
    ((t(3, 4), t(4, dtype=torch.uint8), t(3, dtype=I)), "CUDA"),
])
def test_action_log_prob_refuses(args, text):
    with pytest.raises(ValueError, match=text):
        P.action_log_prob(*args)


def _drafts(**kw):
    a = dict(logits=t(2, 3, 5), drafts=t(2, 2, dtype=I), accept_u=t(2, 2), sample_u=t(2))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(logits=t(2, 5)), "logits"),
    (dict(logits=t(2, 0, 5), drafts=t(2, 0, dtype=I), accept_u=t(2, 0)), "places"),
    (dict(logits=t(2, N.POLICY_MAX_DRAFTS + 2, 1)), "places"),
    (dict(drafts=t(2, 3, dtype=I)), "drafts must be"),
    (dict(drafts=t(2, 2)), "whole numbers"),
    (dict(accept_u=t(2, 3)), "accept_u"),
    (dict(accept_u=t(2, 2, dtype=torch.float64)), "accept_u"),
    (dict(sample_u=t(2, 1)), "sample_u"),
    (dict(draft_logits=t(2, 3, 5)), "draft_logits"),
    (dict(draft_logits=t(2, 2, 5, dtype=H)), "draft_logits"),
    (dict(lengths=t(3, dtype=I)), "lengths must be"),
    (dict(lengths=t(2)), "whole numbers"),
    (dict(mask=t(2, 2, 5, dtype=torch.bool)), "does not fit"),
    (dict(mask=t(2, 3, 5, dtype=I)), "mask must be"),
    (dict(), "CUDA"),
])
def test_verify_drafts_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        P.verify_drafts(**_drafts(**kw))


@pytest.mark.parametrize("args,text", [
    ((t(3, 4), None, t(4)), "u must be"),
    ((t(3, 4), None, t(3, dtype=H)), "u must be"),
    ((t(3, 4), t(3, 1, 4, dtype=torch.bool), t(3)), "does not fit"),
    ((t(3, 4, dtype=I), None, t(3)), "float32"),
    ((t(3, 4), None, t(3)), "CUDA"),
])
def test_sample_actions_refuses(args, text):
    with pytest.raises(ValueError, match=text):
        P.sample_actions(*args)


def _status(name, *args):
    return getattr(N.lib(), name)(*args), N.lib().jq_last_error().decode()


def test_entry_points_refuse_before_they_launch():
    """Status codes of bad arguments; no device is touched (there need not be one)."""
    p = 1 << 20  # an address that is never read: the checks come first
    ln = lambda **k: _status("jq_layer_norm", *({**dict(x=p, xs=8, w=p, b=p, rows=4, dim=8, dt=0, wt=0, eps=1e-5, y=p,  # noqa: E731
                                                        st=p, s=None), **k}).values())
    for k, text in ((dict(x=None), "at least one row"), (dict(rows=0), "at least one row"), (dict(dim=0), "at least"),
                    (dict(dt=3), "dtype"), (dict(dt=1, wt=2), "weights are"), (dict(xs=-1), "stride"),
                    (dict(y=None), "output"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")):
        st, msg = ln(**k)
        assert st == 1 and text in msg, (k, st, msg)
    for k in (dict(rows=2 ** 31), dict(dim=2 ** 30 + 1)):
        st, msg = ln(**k)
        assert st == 4 and "more than" in msg, (k, st, msg)
    lp = lambda **k: _status("jq_action_log_prob", *({**dict(x=p, xs=8, dt=0, m=p, ms=8, a=p, rows=4, n=8, lp=p, e=p,  # noqa: E731
                                                             st=p, bits=p, s=None), **k}).values())
    for k, want, text in ((dict(x=None), 1, "at least one row"), (dict(rows=0), 1, "at least"), (dict(n=0), 1, "at least"),
                          (dict(n=N.POLICY_MAX_ACTIONS + 1), 4, "JQ_POLICY_MAX_ACTIONS"), (dict(rows=2 ** 31), 4, "rows"),
                          (dict(dt=7), 1, "dtype"), (dict(a=None), 1, "missing"), (dict(lp=None), 1, "missing"),
                          (dict(ms=-1), 1, "mask stride"), (dict(st=p + 4), 1, "aligned"), (dict(x=p + 2), 1, "misaligned")):
        st, msg = lp(**k)
        assert st == want and text in msg, (k, st, msg)
    good = dict(games=2, drafts=1, actions=8, dtype=0, logits=p, logits_game=16, logits_place=8, drafted=p, accept_u=p,
                sample_u=p, accepted=p, out_actions=p, log_probs=p)
    for k, want, text in ((dict(games=0), 1, "at least one game"), (dict(drafts=-1), 1, "at least"),
                          (dict(drafts=N.POLICY_MAX_DRAFTS + 1), 4, "JQ_POLICY_MAX_DRAFTS"), (dict(drafted=None), 1, "missing"),
                          (dict(sample_u=None), 1, "missing"), (dict(log_probs=None), 1, "missing"),
                          (dict(mask_place=-1), 1, "stride"), (dict(out_actions=p + 2), 1, "aligned"),
                          (dict(actions=0), 1, "at least"), (dict(draft_logits=p + 2), 1, "aligned")):
        st, msg = _status("jq_verify_drafts", ctypes.byref(N.JqDrafts(**{**good, **k})), None)
        assert st == want and text in msg, (k, st, msg)


def test_drafts_struct_follows_the_header():
    text = (ROOT / "include" / "jq.h").read_text()
    body = text[text.index("typedef struct jq_drafts {"):text.index("} jq_drafts;")].split("{", 1)[1]
    names = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        decl = decl.strip()
        if decl:
            first, *more = decl.split(",")
            names += [re.sub(r"\W", "", x.split()[-1]) for x in [first, *more]]
    assert names == [n for n, _ in N.JqDrafts._fields_]
    assert f"(1 << {N.POLICY_MAX_ACTIONS.bit_length() - 1})" in text and str(N.POLICY_MAX_DRAFTS) in text
