"""The policy operators at the ends of what they take: logits far from zero and far apart, derivatives of more than
one order, rows of one or two places by the million, large constant rows."""
from __future__ import annotations

import pytest
import torch

from junqi_b200 import policy as P
from tests.test_gpu_policy import DTYPES, U, check_norm, check_verify, gen, within

pytestmark = pytest.mark.gpu


# -- logits of any size --------------------------------------------------------------

@pytest.mark.parametrize("n,density", [(40, 0.6), (40, None), (2000, 0.7), (3000, None), (16641, 0.01), (16641, None)])
@pytest.mark.parametrize("top", [2.2e9, 3e9, 8.6e9, 1e10, 6e8, 1.2e9, 2.0 ** 31, 2.0 ** 33, 5e12])
def test_choices_among_logits_far_from_zero(top, n, density):
    """Distances from the largest logit on both sides of 700, beyond which a weight is 0, of positive and of negative logits
    (multiples of 64 or more, so none lies between 700 and 745, where the 64-bit exponential is not yet 0; a place that is
    not one of the largest has a probability below 2^-360)."""
    g = gen(int(top) % 1009 + n)
    games, d = 12, 3
    apart = torch.tensor([0, 256, 512, 640, 768, 832, 1024, 1280, 2048, 4096], device="cuda")
    at = torch.randint(0, 10, (2, games, d + 1, n), generator=g, device="cuda")
    sign = torch.where(torch.arange(games, device="cuda") % 2 == 0, 1.0, -1.0).double()[:, None, None]
    x, y = ((sign * top - apart[k].double()).float() for k in at)
    y = y[:, :d].contiguous()
    mask = None if density is None else torch.rand(games, d + 1, n, generator=g, device="cuda") < density
    best = x[:, :d] if mask is None else x[:, :d].masked_fill(~mask[:, :d], -torch.inf)
    a = best.argmax(-1)
    a[::3] = torch.randint(0, n, (len(a[::3]), d), generator=g, device="cuda")
    au = 0.01 + 0.9 * torch.rand(games, d, generator=g, device="cuda")
    su = torch.rand(games, generator=g, device="cuda")
    check_verify(x, a, au, su, y, mask)
    check_verify(x, a, au, su, None, mask)
    check_verify(x[:, :1], a[:, :0], au[:, :0], su, None, None if mask is None else mask[:, :1])
    s, lp = P.sample_actions(x, mask, torch.rand(games, d + 1, generator=g, device="cuda"))
    legal = torch.ones_like(x, dtype=torch.bool) if mask is None else mask
    some = legal.any(-1)
    peak = x.masked_fill(~legal, -torch.inf).amax(-1)
    assert torch.equal(s >= 0, some)
    assert torch.equal(x.gather(2, s.clamp(min=0).long()[..., None])[..., 0][some], peak[some]), "not one of the largest"
    ties = ((x == peak[..., None]) & legal).sum(-1)
    within(lp[some], -ties[some].double().log(), 20 * U, "log_probs")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,masked", [(100, True), (100, False), (1500, True), (1500, False)])
def test_choices_among_extreme_logits(dtype, n, masked):
    """Legal places at -inf, at the type's lowest and highest values, all equal, and far apart."""
    big = torch.finfo(dtype).max
    x, y = (torch.randn(9, 3, n, generator=gen(s), device="cuda") for s in (4, 5))
    x[0, :, :n // 2] = -torch.inf
    x[1] = -torch.inf
    x[2] = -big
    x[3] = -big
    x[3, :, 7] = 1.0
    x[4] = 5.0
    x[5, :, 10] = big
    x[6, :, 20:] = -big
    x[7] *= 1000
    x[8], y[8] = big, -big
    y[0], y[5] = -big, y[5].clone().index_fill_(1, torch.tensor([3], device="cuda"), big)
    x, y = x.to(dtype), y[:, :2].to(dtype)
    a = x[:, :2].argmax(-1)
    a[::2, 1] = 10
    au = torch.rand(9, 2, generator=gen(6), device="cuda").clamp(min=0.01)
    su = torch.rand(9, generator=gen(7), device="cuda")
    mask = torch.rand(9, 3, n, generator=gen(8), device="cuda") < 0.8 if masked else None
    check_verify(x, a, au, su, y, mask)
    check_verify(x, a, au, su, None, mask)
    check_verify(x[:, :1], a[:, :0], au[:, :0], su, None, None if mask is None else mask[:, :1])


# -- derivatives ---------------------------------------------------------------------------

SHAPES = {"rows": lambda t: t, "boards": lambda t: t.view(2, 3, 8), "one": lambda t: t[0], "columns": lambda t: t.view(8, 6).t(),
          "slice": lambda t: t[:, 1:7], "repeated": lambda t: t[:1].expand(4, 8), "four axes": lambda t: t.view(1, 3, 2, 8)}


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("op", ["norm", "logp", "entropy"])
def test_second_derivatives_are_refused_whatever_the_shape(op, shape):
    """A gradient that enters a penalty: its own derivative is an error, never left out of the sum."""
    base = torch.randn(6, 8, generator=gen(1), device="cuda")
    x = SHAPES[shape](base).detach()
    if shape != "repeated":
        x.requires_grad_(True)
        leaf = x
    else:
        leaf = base[:1].clone().requires_grad_(True)
        x = leaf.expand(4, 8)
    if op == "norm":
        loss = P.layer_norm(x, torch.ones(x.shape[-1], device="cuda")).square().sum()
    else:
        m = torch.rand(x.shape[-1], generator=gen(2), device="cuda") < 0.8
        out = P.action_log_prob(x, m, torch.zeros(x.shape[:-1], dtype=torch.int32, device="cuda"))
        loss = out[0 if op == "logp" else 1].sum()
    (g,) = torch.autograd.grad(loss, leaf, create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(loss + g.square().sum(), leaf)


@pytest.mark.parametrize("which", ["weight", "bias", "dy", "x of a linear layer"])
def test_second_derivatives_of_the_other_inputs_are_refused(which):
    x = torch.randn(2, 3, 8, generator=gen(1), device="cuda")
    w, b = (torch.rand(8, generator=gen(s), device="cuda") for s in (2, 3))
    dy = torch.randn(2, 3, 8, generator=gen(4), device="cuda")
    lin = torch.rand(8, 8, generator=gen(5), device="cuda", requires_grad=True)
    leaf = {"weight": w, "bias": b, "dy": dy, "x of a linear layer": lin}[which].requires_grad_(True)
    h = x @ lin
    y = P.layer_norm(h, w, b)
    wrt = [v for v in (h, w, b) if v.requires_grad]
    if which == "dy":
        x.requires_grad_(True)
        wrt, y = [x], P.layer_norm(x, w, b)
    if which == "bias":  # no gradient depends on it, so there is nothing to refuse
        (g,) = torch.autograd.grad(y, b, dy, create_graph=True)
        return within(g, dy.double().sum((0, 1)), 8 * U * dy.abs().sum((0, 1)).double(), "db")
    grads = torch.autograd.grad(y, wrt, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(sum(g.square().sum() for g in grads), leaf)


# -- layer norm's layouts -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 2, 4, 7, 16])
def test_layer_norm_short_rows_by_the_million(dtype, dim):
    rows = 3_000_017
    g = gen(dim)
    x, dy = (torch.randn(rows, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    w, b = (torch.rand(dim, generator=g, device="cuda") for _ in range(2))
    check_norm(x, w, b, dy)
    wide = torch.randn(rows, dim + 3, generator=g, device="cuda").to(dtype)
    check_norm(wide[:, 1:1 + dim], w, None, dy)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [60, 200, 708, 1111, 2047, 7356, 8191, 9001])
def test_layer_norm_large_constant_rows(dtype, dim):
    """A row of one number has no spread: its result is the bias whatever the number, and its gradients are those of a row
    of zeros (a mean in 64 bits would not show it: rounded, it misses a number of 24 bits of that size by more than eps).
    Beside them rows of two neighbouring numbers, and large numbers whose squares overflow."""
    rows = 400
    g = gen(dim)
    x = (10 ** (3 + 15 * torch.rand(rows, 1, generator=g, device="cuda", dtype=torch.float64))).to(dtype)
    x = x * torch.where(torch.arange(rows, device="cuda") % 2 == 0, 1, -1).to(dtype)[:, None]
    x[0], x[1], x[2] = 3e33, -1e34, 1e38 / dim
    x = x.expand(rows, dim).contiguous()
    w, b = (torch.rand(dim, generator=g, device="cuda") for _ in range(2))
    dy = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    z = x.requires_grad_(True)
    o = torch.zeros_like(x).requires_grad_(True)
    w.requires_grad_(True)
    b.requires_grad_(True)
    y = P.layer_norm(z, w, b)
    assert torch.equal(y, b.to(dtype).expand(rows, dim))
    of_zeros = torch.autograd.grad(P.layer_norm(o, w, b), (o, w, b), dy)
    for got, want in zip(torch.autograd.grad(y, (z, w, b), dy), of_zeros):
        assert torch.equal(got, want)
    x = x.detach()
    check_norm(torch.zeros_like(x), w, b, dy)
    if dtype == torch.float32:
        big = x[:, :1].clamp(-1e12, 1e12).clone()
        two = torch.where(torch.rand(rows, dim, generator=g, device="cuda") < 0.5, big, torch.nextafter(big, 2 * big))
        check_norm(two, w, b, dy)


# -- kept drafts without a mask ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("games,n", [(1, 262144), (64, 40000), (700, 262144), (700, 16641), (640, 33)])
def test_log_probabilities_of_kept_drafts_of_any_number_of_games(games, n, dtype):
    """Their log Z is of 32 bits: an exponential is off by 4 u, its argument's three roundings by 3 * 18 u on average (log2 n
    <= 18), nine additions before a sum joins its lane's; a lane has at most n / 256 of those (eight places or more each), whose
    addition and factor for a risen maximum cost 6 u; five joins of 5 u.  With 700 games a row is one CTA's.  Rising rows
    raise the maximum at every step."""
    g = gen(games + n)
    x = torch.randn(games, 2, n, generator=g, device="cuda").mul_(2)
    x[0::4, 0] = torch.linspace(-6, 3, n, device="cuda")
    x[1::4, 0] = torch.linspace(4, -5, n, device="cuda")
    x[2::4, 0] = -0.3
    x = x.to(dtype)
    a = torch.randint(0, n, (games, 1), generator=g, device="cuda")
    v = P.verify_drafts(x, a, torch.zeros(games, 1, device="cuda"), torch.rand(games, generator=g, device="cuda"))
    assert (v.accepted == 1).all() and torch.equal(v.actions[:, :1].long(), a)
    for k in range(0, games, 100):
        xd = x[k:k + 100, 0].double()
        want = xd.gather(1, a[k:k + 100])[:, 0] - xd.logsumexp(1)
        within(v.log_probs[k:k + 100, 0], want, 1.01 * (92 + 6 * max(n / 256, 1) + want.abs()) * U, "log_probs")


# -- tensors that are negated when they are read ------------------------------------------------------

def lazily_negated(t):
    """t, as the imaginary part of a conjugate: memory holds -t, and a bit says so."""
    v = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert v.is_neg() and torch.equal(v.resolve_neg(), t)
    return v


@pytest.mark.parametrize("n", [1, 30])
def test_lazily_negated_inputs(n):
    x, w, b, dy = (torch.randn(s, generator=gen(k), device="cuda") for k, s in enumerate([(5, n), (n,), (n,), (5, n)]))
    lazy = lazily_negated

    def norm(x, w, b, dy):
        x, w, b = (v.detach().requires_grad_(True) for v in (x, w, b))
        y = P.layer_norm(x, w, b)
        with torch.no_grad():
            assert torch.equal(y, P.layer_norm(x, w, b))
        return y, *torch.autograd.grad(y, (x, w, b), dy)

    for got, want in zip(norm(lazy(x), lazy(w), lazy(b), lazy(dy)), norm(x, w, b, dy)):
        assert torch.equal(got, want)
    a = torch.randint(0, n, (5,), generator=gen(7), device="cuda")
    u, r = (torch.rand(5, generator=gen(s), device="cuda") for s in (8, 9))

    def logp(x, u, r):
        x = x.detach().requires_grad_(True)
        out = P.action_log_prob(x, None, a)
        return *out, *torch.autograd.grad(out, x, (u, r)), *P.action_log_prob(x.detach(), None, a)

    for k in (slice(0, 5), slice(0, 1)):
        for got, want in zip(P.sample_actions(lazy(x[k]), None, lazy(r[k])), P.sample_actions(x[k], None, r[k])):
            assert torch.equal(got, want)
        x2, y2 = x[k, None].expand(-1, 2, -1).contiguous(), dy[k, None].contiguous()
        for got, want in zip(P.verify_drafts(lazy(x2), a[k, None], lazy(u[k, None]), lazy(r[k]), draft_logits=lazy(y2)),
                             P.verify_drafts(x2, a[k, None], u[k, None], r[k], draft_logits=y2)):
            assert torch.equal(got, want)
    for got, want in zip(logp(lazy(x), lazy(u), lazy(r)), logp(x, u, r)):
        assert torch.equal(got, want)


def test_gradients_through_a_conjugate():
    """What torch hands to the backward pass of a value that went into a complex number."""
    x = torch.randn(6, 20, generator=gen(1), device="cuda", requires_grad=True)
    a = torch.randint(0, 20, (6,), generator=gen(2), device="cuda")
    c = torch.randn(6, generator=gen(3), device="cuda")
    for op in (lambda: P.action_log_prob(x, None, a)[0], lambda: P.action_log_prob(x, None, a)[1], lambda: P.layer_norm(x)[:, 3]):
        v = op()
        (got,) = torch.autograd.grad((torch.complex(torch.zeros_like(v), v).conj().imag * c).sum(), x)
        (want,) = torch.autograd.grad((op() * -c).sum(), x)
        assert torch.equal(got, want)
