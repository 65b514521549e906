"""The policy operators' cases: layer norm of a policy's features, log-probability and entropy of actions under a legal
mask, and verification of drafted actions (with no drafts: sampling), each with its plain form in torch.

`own` chooses what `run` calls: False, the plain forms below; True, `junqi_b200.policy`.
"""
import math

import torch

own = False

ACTIONS = 16641  # canonical actions: 129 source cells x 129 destination cells
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
RESIDUAL_MIN = 2.0 ** -40  # verification: less probability left after a rejection counts as none
EPS = 1e-5


def listed():
    return [
        # One ply's features of a few environments, while acting: latency.
        {"name": "norm_act_64x512_bf16", "op": "norm", "rows": 64, "dim": 512, "dtype": "bf16", "weights": "fp32", "pad": 0, "grad": False},
        # A training minibatch of 2,048 positions, one token for each of the 129 board cells.
        {"name": "norm_train_264192x256_bf16", "op": "norm", "rows": 2048 * 129, "dim": 256, "dtype": "bf16", "weights": "fp32", "pad": 0, "grad": True},
        # A trunk's features of a minibatch in full precision, an odd width whose rows start anywhere.
        {"name": "norm_train_8191x1111_fp32", "op": "norm", "rows": 8191, "dim": 1111, "dtype": "fp32", "weights": "fp32", "pad": 0, "grad": True},
        # Wide features, a slice of a wider buffer.
        {"name": "norm_train_6000x4096_fp16", "op": "norm", "rows": 6000, "dim": 4096, "dtype": "fp16", "weights": "fp16", "pad": 64, "grad": True},
        # The score of one position's action in 16 games: latency.
        {"name": "logp_eval_16_fp32", "op": "logp", "rows": 16, "actions": ACTIONS, "dtype": "fp32", "legal": 80, "pad": 0, "grad": False},
        # A training minibatch of 4,096 plies, logits as a matrix product leaves them when its columns are padded.
        {"name": "logp_train_4096_bf16", "op": "logp", "rows": 4096, "actions": ACTIONS, "dtype": "bf16", "legal": 80, "pad": 7, "grad": True},
        # A larger one in full precision, with crowded late boards among its legal sets.
        {"name": "logp_train_8192_fp32", "op": "logp", "rows": 8192, "actions": ACTIONS, "dtype": "fp32", "legal": 400, "pad": 0, "grad": True},
        # No mask: a belief or imitation head over a plain vocabulary.
        {"name": "logp_train_2048x30001_fp16", "op": "logp", "rows": 2048, "actions": 30001, "dtype": "fp16", "legal": 0, "pad": 0, "grad": True},
        # Every ply of a rollout: 4,096 environments draw one action each.
        {"name": "sample_4096_fp32", "op": "verify", "games": 4096, "drafts": 0, "actions": ACTIONS, "dtype": "fp32", "legal": 80, "scored": True, "ragged": False},
        # Eight evaluation games with four drafted plies each: latency.
        {"name": "verify_8x4_bf16", "op": "verify", "games": 8, "drafts": 4, "actions": ACTIONS, "dtype": "bf16", "legal": 80, "scored": True, "ragged": False},
        # Many games, eight drafted plies, of which some games use fewer.
        {"name": "verify_1024x8_fp32", "op": "verify", "games": 1024, "drafts": 8, "actions": ACTIONS, "dtype": "fp32", "legal": 120, "scored": True, "ragged": True},
        # No mask: drafts from another network over a plain vocabulary.
        {"name": "verify_301x5_nomask_bf16", "op": "verify", "games": 301, "drafts": 5, "actions": ACTIONS, "dtype": "bf16", "legal": 0, "scored": True, "ragged": True},
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    op = rng.choice(["norm", "logp", "verify"])
    if op == "norm":
        dim = _between(rng, 28, 8192)
        rows = min(_between(rng, 1, 262144), 2048 * 129 * 256 * 2 // (dim * size))
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "weights": rng.choice(["fp32", dtype]),
                "pad": rng.choice([0, 0, 8, 5]), "grad": rng.random() < 0.7}
    actions = rng.choice([ACTIONS, ACTIONS, _between(rng, 129, 50000)])
    legal = rng.choice([_between(rng, 1, 512), _between(rng, 1, 512), 0])
    legal = min(legal, actions)
    if op == "logp":
        rows = min(_between(rng, 1, 8192), 8192 * ACTIONS * 4 // (actions * size) // (4 if legal == 0 else 1))
        return {"op": op, "rows": rows, "actions": actions, "dtype": dtype, "legal": legal,
                "pad": rng.choice([0, 0, (-actions) % 8]), "grad": rng.random() < 0.7}
    drafts = rng.choice([0, 1, 2, 3, 4, 5, 6, 8, 11])
    games = min(_between(rng, 1, 1024), 1024 * 8 * ACTIONS // (max(1, drafts) * actions) // (4 if legal == 0 else 1))
    return {"op": op, "games": games, "drafts": drafts, "actions": actions, "dtype": dtype, "legal": legal,
            "scored": rng.random() < 0.7, "ragged": rng.random() < 0.5}


def _legal_mask(rows, actions, legal, gen):
    """(rows, actions) uint8: up to `legal` legal places a row, one row in 61 without any (a finished game)."""
    dev = gen.device
    count = torch.randint(max(1, legal // 4), legal + 1, (rows, 1), generator=gen, device=dev)
    count[torch.randint(0, 61, (rows, 1), generator=gen, device=dev) == 0] = 0
    place = torch.randint(0, actions, (rows, legal), generator=gen, device=dev)
    on = torch.arange(legal, device=dev)[None, :] < count
    mask = torch.zeros((rows, actions + 1), dtype=torch.uint8, device=dev)
    mask.scatter_(1, torch.where(on, place, actions), 1)
    return mask[:, :actions].contiguous()


def _pick(scores, mask, gen):
    """An action of each row's softmax (Gumbel-max), -1 where the mask leaves none."""
    x = scores.float()
    g = -torch.log(-torch.log(torch.rand(x.shape, generator=gen, device=x.device).clamp_(1e-12, 1 - 1e-7)))
    x = x + g
    if mask is not None:
        x = x.masked_fill(mask == 0, -math.inf)
    a = x.argmax(-1).to(torch.int32)
    return a if mask is None else torch.where((mask != 0).any(-1), a, -1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 11)
    dev, dt = gen.device, DTYPES[case["dtype"]]
    normal = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    s = {"op": case["op"], "grad": case.get("grad", False)}
    if case["op"] == "norm":
        rows, dim, wt = case["rows"], case["dim"], DTYPES[case["weights"]]
        # features with a mean and a spread of their own in each row
        x = normal(rows, dim + case["pad"]).mul_(0.5 + normal(rows, 1).abs()).add_(normal(rows, 1)).to(dt)
        s |= {"x": x[:, :dim], "weight": (1 + 0.1 * normal(dim)).to(wt), "bias": (0.1 * normal(dim)).to(wt)}
        if s["grad"]:
            s |= {"dy": normal(rows, dim).to(dt)}
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_(True)
        return s
    actions, legal = case["actions"], case["legal"]
    if case["op"] == "logp":
        rows = case["rows"]
        x = normal(rows, actions + case["pad"]).mul_(2.0).to(dt)[:, :actions]
        mask = _legal_mask(rows, actions, legal, gen) if legal else None
        s |= {"logits": x, "mask": mask, "actions": _pick(x, mask, gen)}
        if s["grad"]:
            scale = 1.0 if dt == torch.float16 else 1 / rows  # a mean's gradient; with fp16, its loss scaled up
            s |= {"g_lp": normal(rows) * scale, "g_ent": torch.full((rows,), -0.01 * scale, device=dev)}
            s["logits"].requires_grad_(True)
        return s
    games, drafts = case["games"], case["drafts"]
    target = normal(games, drafts + 1, actions).mul_(2.0)
    near = target[:, :drafts] + 0.4 * normal(games, drafts, actions)
    mask = _legal_mask(games * (drafts + 1), actions, legal, gen).view(games, drafts + 1, actions) if legal else None
    near = near.to(dt)
    s |= {"logits": target.to(dt), "mask": mask, "drafts": _pick(near, None if mask is None else mask[:, :drafts], gen),
          "draft_logits": near if case["scored"] and drafts else None,
          "lengths": torch.randint(0, drafts + 1, (games,), generator=gen, device=dev, dtype=torch.int32) if case["ragged"] else None,
          "accept": torch.rand((games, drafts), generator=gen, device=dev), "draw": torch.rand((games,), generator=gen, device=dev)}
    return s


# ---- plain forms -----------------------------------------------------------

def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    d = x.shape[1]
    c = x - x.mean(1, keepdim=True)
    c = c - c.mean(1, keepdim=True)  # what the first mean's rounding left
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    xh = c * r
    y = (xh * w + b).to(s["x"].dtype)
    if not s["grad"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.sum(1, keepdim=True) / d - xh * ((g * xh).sum(1, keepdim=True) / d))
    dw, db = (dy * xh).sum(0, dtype=torch.float64), dy.sum(0, dtype=torch.float64)
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": dw.to(s["weight"].dtype), "db": db.to(s["bias"].dtype)}


def _plain_softmax(x, mask):
    """(shifted logits, e, Z, empty row) over the legal places of the last axis, in x's type."""
    if mask is not None:
        x = torch.where(mask != 0, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    empty = m == -math.inf
    c = x - torch.where(empty, 0.0, m)
    e = torch.exp(c)
    return c, e, e.sum(-1, keepdim=True), empty


def _plain_logp(s):
    c, e, z, empty = _plain_softmax(s["logits"].float(), s["mask"])
    z = torch.where(empty, 1.0, z)
    logz, p = torch.log(z), e / z
    a = s["actions"].long()[:, None]
    inside = (a >= 0) & (a < c.shape[1])
    at = a.clamp(0, c.shape[1] - 1)
    ca = c.gather(1, at)
    lp = torch.where(inside, ca - logz, 0.0)
    ent = torch.where(empty, 0.0, logz - torch.where(e > 0, p * c, 0.0).sum(1, keepdim=True))
    out = {"log_prob": lp[:, 0], "entropy": ent[:, 0]}
    if s["grad"]:
        glp = torch.where(inside & (ca > -math.inf), s["g_lp"][:, None], 0.0)
        dx = torch.where(e > 0, -p * (glp + s["g_ent"][:, None] * (c - logz + ent)), 0.0)
        dx.scatter_add_(1, at, glp)
        out["dlogits"] = dx.to(s["logits"].dtype)
    return out


def _plain_verify(s):
    # whole numbers come out, so the borders are computed in 64 bits
    games, places, actions = s["logits"].shape
    drafts = places - 1
    c, e, z, empty = _plain_softmax(s["logits"].double(), s["mask"])
    z = torch.where(empty, 1.0, z)
    p = e / z
    a = s["drafts"].long()
    inside = (a >= 0) & (a < actions)
    at = a.clamp(0, actions - 1)[..., None]
    if s["draft_logits"] is not None:
        _, eq, zq, none = _plain_softmax(s["draft_logits"].double(), None if s["mask"] is None else s["mask"][:, :drafts])
        q = eq / torch.where(none, 1.0, zq)
    else:
        q = torch.zeros_like(p[:, :drafts]).scatter_(2, at, inside[..., None].double())
    n = s["lengths"].long() if s["lengths"] is not None else torch.full((games,), drafts, device=p.device)
    step = torch.arange(drafts, device=p.device)[None, :]
    pa, qa = p[:, :drafts].gather(2, at)[..., 0], q.gather(2, at)[..., 0]
    keep = inside & (s["accept"].double() * qa < pa) & (step < n[:, None])
    accepted = keep.long().cumprod(1).sum(1)
    row = torch.arange(games, device=p.device)
    pr = p[row, accepted]
    q = torch.cat([q, torch.zeros_like(p[:, :1])], 1)
    w = (pr - torch.where((accepted < n)[:, None], q[row, accepted], 0.0)).clamp(min=0)
    w = torch.where(w.sum(1, keepdim=True) > RESIDUAL_MIN, w, pr)
    run = w.cumsum(1)
    over = run > s["draw"].double()[:, None] * run[:, -1:]
    places_of = torch.arange(actions, device=p.device)
    last = torch.where(w > 0, places_of, -1).amax(1)
    first = torch.where(over, places_of, actions).amin(1)
    nxt = torch.where(first < actions, first, last)
    out = torch.cat([a, torch.full((games, 1), -1, device=p.device)], 1)
    step = torch.arange(places, device=p.device)[None, :]
    out = torch.where(step < accepted[:, None], out, torch.where(step == accepted[:, None], nxt[:, None], -1))
    lp = (c - torch.log(z)).gather(2, out.clamp(min=0)[..., None])[..., 0]
    lp = torch.where(out >= 0, lp, 0.0).float()
    if drafts == 0:
        return {"actions": out[:, 0].to(torch.int32), "log_probs": lp[:, 0]}
    return {"accepted": accepted.to(torch.int32), "actions": out.to(torch.int32), "log_probs": lp}


def run(state):
    s = state
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "logp": _plain_logp, "verify": _plain_verify}[s["op"]](s)
    from junqi_b200 import policy
    if s["op"] == "norm":
        y = policy.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        if not s["grad"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if s["op"] == "logp":
        lp, ent = policy.action_log_prob(s["logits"], s["mask"], s["actions"])
        if not s["grad"]:
            return {"log_prob": lp, "entropy": ent}
        (dx,) = torch.autograd.grad((lp, ent), (s["logits"],), (s["g_lp"], s["g_ent"]))
        return {"log_prob": lp.detach(), "entropy": ent.detach(), "dlogits": dx}
    if s["drafts"].shape[1] == 0:
        actions, lp = policy.sample_actions(s["logits"][:, 0], None if s["mask"] is None else s["mask"][:, 0], s["draw"])
        return {"actions": actions, "log_probs": lp}
    v = policy.verify_drafts(s["logits"], s["drafts"], s["accept"], s["draw"], draft_logits=s["draft_logits"],
                             mask=s["mask"], lengths=s["lengths"])
    return {"accepted": v.accepted, "actions": v.actions, "log_probs": v.log_probs}


def _seen(case):
    """Legal places of a row that have to be read: on average 5/8 of the most, all without a mask."""
    return 0.625 * case["legal"] * 60 / 61 if case["legal"] else case["actions"]


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        n, d, w = case["rows"] * case["dim"], case["dim"], DTYPES[case["weights"]].itemsize
        if not case["grad"]:
            return {"bytes": 2 * n * size + 2 * d * w, "flops": 8 * n}
        # forward: x in, y out; backward: x and dy in, dx out, with the weights' gradients
        return {"bytes": 5 * n * size + 5 * d * w, "flops": 22 * n}
    seen, masked = _seen(case), case["actions"] if case["legal"] else 0
    if case["op"] == "logp":
        rows = case["rows"]
        fwd = rows * (masked + seen * size + 4 + 8)
        if not case["grad"]:
            return {"bytes": fwd, "flops": 6 * rows * seen}
        return {"bytes": fwd + rows * (seen * size + 8 + case["actions"] * size), "flops": 14 * rows * seen}
    # a game is read up to its first rejection: a scored draft is kept about 6 times in 7, a bare one once in 4 (both as `prepare` makes them)
    keep = 0.86 if case["scored"] else 0.23
    n = case["drafts"] / 2 if case["ragged"] else case["drafts"]
    places = (1 - keep ** (n + 1)) / (1 - keep)
    rows = places * (1 + (1 if case["scored"] and n else 0))
    games = case["games"]
    return {"bytes": games * (places * masked + rows * seen * size + 8 * n + 4 + 8 * (case["drafts"] + 1) + 4),
            "flops": 8 * games * rows * seen}


# ---- from the definitions, in 64 bits --------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "norm":
        x, w, b = (s[k].detach().double().requires_grad_(True) for k in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) * (var + EPS).rsqrt() * w + b
        if not s["grad"]:
            return {"y": y.detach()}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    x = s["logits"].detach().double()
    legal = torch.ones(x.shape, dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"].bool()
    if s["op"] == "logp":
        x.requires_grad_(True)
        some = legal.any(1)
        # an empty row takes part as a row of one place, and is taken out again
        lse = torch.logsumexp(torch.where(legal | ~some[:, None] & (torch.arange(x.shape[1], device=x.device) == 0), x, -math.inf), 1)
        logp = x - lse[:, None]
        a = s["actions"].long()
        real = (a >= 0) & (a < x.shape[1])
        at = a.clamp(0, x.shape[1] - 1)[:, None]
        lp = torch.where(real & legal.gather(1, at)[:, 0], logp.gather(1, at)[:, 0], torch.where(real, -math.inf, 0.0))
        ent = torch.where(some, -torch.where(legal, logp.exp() * logp, 0.0).sum(1), 0.0)
        if not s["grad"]:
            return {"log_prob": lp.detach(), "entropy": ent.detach()}
        (dx,) = torch.autograd.grad((lp, ent), (x,), (s["g_lp"].double(), s["g_ent"].double()))
        return {"log_prob": lp.detach(), "entropy": ent.detach(), "dlogits": dx}
    games, places, _ = x.shape
    if games * places * case["actions"] > 2 ** 28:
        return None
    logp = torch.log_softmax(x.masked_fill(~legal, -math.inf), 2)
    p = torch.where(legal, logp.exp(), 0.0)
    logq = None
    if s["draft_logits"] is not None:
        logq = torch.log_softmax(s["draft_logits"].double().masked_fill(~legal[:, :places - 1], -math.inf), 2)
    drafts, lengths = s["drafts"].cpu().tolist(), (None if s["lengths"] is None else s["lengths"].cpu().tolist())
    accept, point = s["accept"].double().cpu().tolist(), s["draw"].double()
    pa = p[:, :places - 1].gather(2, s["drafts"].long().clamp(min=0)[..., None])[..., 0].cpu().tolist()
    qa = None if logq is None else logq.exp().nan_to_num(0.0).gather(2, s["drafts"].long().clamp(min=0)[..., None])[..., 0].cpu().tolist()
    kept, left = [], []
    for g in range(games):
        n, i = places - 1 if lengths is None else lengths[g], 0
        while i < n and drafts[g][i] >= 0 and accept[g][i] * (1.0 if qa is None else qa[g][i]) < pa[g][i]:
            i += 1
        kept.append(i)
        left.append(i < n)
    kept_t = torch.tensor(kept, device=x.device)
    games_t = torch.arange(games, device=x.device)
    weights = p[games_t, kept_t].clone()
    cut = torch.tensor(left, device=x.device)
    if places > 1:
        at = kept_t.clamp(max=places - 2)
        if logq is not None:
            q = logq[games_t, at].exp().nan_to_num(0.0)
        else:
            a = s["drafts"].long()[games_t, at]
            q = torch.nn.functional.one_hot(a.clamp(min=0), case["actions"]).double() * (a >= 0)[:, None]
        rest = (weights - q).clamp(min=0)
        weights = torch.where((cut & (rest.sum(1) > RESIDUAL_MIN))[:, None], rest, weights)
    edge = weights.cumsum(1)
    nxt = torch.searchsorted(edge, (point * edge[:, -1])[:, None], right=True)[:, 0]
    top = case["actions"] - 1 - (weights.flip(1) > 0).to(torch.int8).argmax(1)
    nxt = torch.where(edge[:, -1] > 0, torch.minimum(nxt, top), -1)
    out = torch.full((games, places), -1, dtype=torch.int64, device=x.device)
    out[:, :places - 1] = s["drafts"].long()
    step = torch.arange(places, device=x.device)[None, :]
    out = torch.where(step < kept_t[:, None], out, torch.where(step == kept_t[:, None], nxt[:, None], -1))
    lp = torch.where(out >= 0, logp.gather(2, out.clamp(min=0)[..., None])[..., 0], 0.0)
    if places == 1:
        return {"actions": out[:, 0].to(torch.int32), "log_probs": lp[:, 0]}
    return {"accepted": kept_t.to(torch.int32), "actions": out.to(torch.int32), "log_probs": lp}
