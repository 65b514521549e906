"""Policy operators against plain implementations in 64 bits.

Tolerances follow from the arithmetic, with u = 2^-24 (half a step of 32
bits) and h = torch.finfo(type).eps / 2 for the result's rounding:

* layer norm: a sum of n values in a thread-and-tree order has at most
  k = n / 512 + 32 roundings on any path (16 places a thread, five or nine
  levels of the tree; the long form n / 512 places a thread), each u of the
  partial sums, which are at most sum |.|.  So xh is off by at most
  (2 k + 8) u (|xh| + 1), and what is made of it accordingly.
* sums over rows: at most `rows` roundings, u of sum |.| each.
* exp of d <= 0 by a base-2 exponential: 2^-22 + |d| u relative (2 units of
  the instruction, and the argument's rounding), so a sum of them is off by
  (n / 256 + 24 + 4 + D) u relative, D the largest -d, and log Z by as much.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from junqi_b200 import policy as P

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def within(got, want, tol, what):
    """|got - want| <= tol wherever want is a number; elsewhere the same infinity or NaN."""
    got, want = got.detach().double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=want.device).expand(want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), f"{what}: infinities differ"
    bad = fin & ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, e.g. {got[bad][:3].tolist()} for "
                           f"{want[bad][:3].tolist()} +- {tol[bad][:3].tolist()}")


def half_step(t, dtype):
    f = torch.finfo(dtype)
    return t.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2  # subnormal results round by a fixed step


# -- layer norm ------------------------------------------------------------------

def check_norm(x, w, b, dy, eps=1e-5, mean=0.0):
    x, w, b = (None if v is None else v.detach().requires_grad_(True) for v in (x, w, b))
    y = P.layer_norm(x, w, b, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(y, P.layer_norm(x, w, b, eps))
    leaves = [v for v in (x, w, b) if v is not None]
    got = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(P.layer_norm(x, w, b, eps), leaves, dy)
    for a, c in zip(got, again):
        assert torch.equal(a, c), "not the same bits twice"

    n = x.shape[-1]
    xd, dyd = x.detach().double().reshape(-1, n), dy.double().reshape(-1, n)
    wd = torch.ones(n, dtype=torch.float64, device="cuda") if w is None else w.detach().double()
    bd = torch.zeros_like(wd) if b is None else b.detach().double()
    mu = xd.mean(1, keepdim=True)
    var = ((xd - mu) ** 2).mean(1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    xh = (xd - mu) * r
    k = 2 * (n / 512 + 32) + 8
    want = xh * wd + bd
    e_xh = k * U * (xh.abs() + 1)
    within(y.reshape(-1, n), want, half_step(want, x.dtype) * 1.001 + 1.01 * (e_xh * wd.abs() + 2 * U * (want.abs() + bd.abs())), "y")
    g = dyd * wd
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - c1 - xh * c2)
    size = r * (g.abs() + g.abs().mean(1, keepdim=True) + (xh.abs() + 1) * ((g.abs() * (xh.abs() + 1)).mean(1, keepdim=True)))
    within(got[0].reshape(-1, n), dx, half_step(dx, x.dtype) * 1.001 + 2 * k * U * size, "dx")
    at = 1
    rows = xd.shape[0]
    for v, terms, name in ((w, dyd * xh, "dw"), (b, dyd, "db")):
        if v is None:
            continue
        want = terms.sum(0)
        err = (rows + 16) * U * terms.abs().sum(0)
        if name == "dw":
            err = err + (dyd.abs() * e_xh).sum(0)
        assert got[at].dtype == v.dtype
        within(got[at], want, half_step(want, v.dtype) * 1.001 + 1.01 * err, name)
        at += 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (5, 1), (3, 2), (1, 8), (70, 28), (33, 31), (9, 64), (300, 129), (17, 250),
                                      (64, 256), (65, 257), (40, 512), (11, 1000), (7, 1111), (6, 2047), (5, 4096),
                                      (3, 4100), (3, 8192), (2, 8193), (3, 20000)])
def test_layer_norm(dtype, rows, dim):
    g = gen(rows * 131 + dim)
    x = torch.randn(rows, dim, generator=g, device="cuda").mul_(1.7).add_(0.4).to(dtype)
    w = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda"))
    b = 0.3 * torch.randn(dim, generator=g, device="cuda")
    dy = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    check_norm(x, w, b, dy)
    check_norm(x, w.to(dtype), b.to(dtype), dy)


def test_layer_norm_many_rows():
    """More rows than the grid holds at once: the walk over the rows and its last, partial step."""
    for rows, dim in ((20011, 24), (9001, 200), (3001, 600)):
        g = gen(rows)
        x = torch.randn(rows, dim, generator=g, device="cuda")
        check_norm(x, torch.rand(dim, generator=g, device="cuda"), None, torch.randn(rows, dim, generator=g, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_without_weights_and_partly(dtype):
    x, dy = (torch.randn(37, 96, generator=gen(s), device="cuda").to(dtype) for s in (1, 2))
    w = torch.rand(96, generator=gen(3), device="cuda")
    check_norm(x, None, None, dy)
    check_norm(x, w, None, dy)
    check_norm(x, None, w.to(dtype), dy)


@pytest.mark.parametrize("dim", [64, 200, 1000])
def test_layer_norm_hard_rows(dim):
    """Constant rows, a large mean, a spread far below eps, and large values, side by side."""
    g = gen(7)
    x = torch.randn(6, dim, generator=g, device="cuda")
    x[1] = 3.25
    x[2] = 0
    x[3] = x[3] + 1000
    x[4] *= 1e-6
    x[5] *= 1e15
    check_norm(x, torch.rand(dim, generator=g, device="cuda"), torch.rand(dim, generator=g, device="cuda"),
               torch.randn(6, dim, generator=g, device="cuda"))


def test_layer_norm_nan_stays_in_its_row():
    x = torch.randn(9, 40, generator=gen(1), device="cuda")
    clean = P.layer_norm(x)
    x[4, 7], x[6, 0] = float("nan"), float("inf")
    y = P.layer_norm(x)
    keep = torch.tensor([0, 1, 2, 3, 5, 7, 8], device="cuda")
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[4]).all() and torch.isnan(y[6]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_strides(dtype):
    """Slices of wider rows (aligned and not), a transposed array, leading axes, repeated and broadcast inputs."""
    g = gen(11)
    wide = torch.randn(24, 300, generator=g, device="cuda").to(dtype)
    w, b = (torch.rand(256, generator=g, device="cuda") for _ in range(2))
    dy = torch.randn(24, 256, generator=g, device="cuda").to(dtype)
    for at in (0, 1, 8, 13):
        check_norm(wide[:, at:at + 256], w, b, dy)
    check_norm(torch.randn(256, 24, generator=g, device="cuda").to(dtype).t(), w, b, dy)
    check_norm(wide[:, :256].reshape(2, 3, 4, 256), w, b, dy.reshape(2, 3, 4, 256))
    check_norm(wide[:1, :256].expand(24, 256), w, b, dy)
    check_norm(wide[:, :256], w, b, dy[:1].expand(24, 256))
    check_norm(wide[:, :256], w, b, dy[0, 0].expand(24, 256))
    check_norm(wide[0, :256], w, b, dy[0])
    check_norm(wide[:, :256], torch.rand(512, generator=g, device="cuda")[::2], b, dy)


def test_layer_norm_shared_leaf_and_broadcast_gradients():
    """One weight in two calls, and features that were broadcast: gradients add up."""
    g = gen(5)
    x = torch.randn(4, 1, 64, generator=g, device="cuda", requires_grad=True)
    w = torch.rand(64, generator=g, device="cuda", requires_grad=True)
    dy = torch.randn(4, 6, 64, generator=g, device="cuda")
    y = P.layer_norm(x.expand(4, 6, 64), w) * dy
    (y.sum() + (P.layer_norm(x, w) * dy[:, :1]).sum()).backward()
    a, v = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)

    def plain(t):
        c = t - t.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * v

    ((plain(a.expand(4, 6, 64)) * dy.double()).sum() + (plain(a) * dy[:, :1].double()).sum()).backward()
    # 7 rows of at most 144 u (|dx| + ...) each; sizes here are below 20
    within(x.grad, a.grad, 7 * 144 * U * 20, "dx")
    within(w.grad, v.grad, 28 * 144 * U * 20, "dw")


def test_layer_norm_gradient_against_differences():
    """Central differences of the operator's own forward pass: its error (72 u of about 3) over the step 2^-6,
    and the third derivative (about 10) times the step squared."""
    g = gen(9)
    x, dy = (torch.randn(3, 20, generator=g, device="cuda") for _ in range(2))
    w = torch.rand(20, generator=g, device="cuda")
    xr = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(P.layer_norm(xr, w), xr, dy)
    h = 2.0 ** -6
    for j in range(0, 20, 3):
        up, dn = x.clone(), x.clone()
        up[:, j] += h
        dn[:, j] -= h
        f = lambda v: (P.layer_norm(v, w).double() * dy.double()).sum(1)  # noqa: E731
        within(dx[:, j], (f(up) - f(dn)) / (2 * h), 20 * 72 * U * 3 * 4 / h + 10 * 20 * h * h, "dx")


def test_layer_norm_empty_batch():
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = P.layer_norm(x, w)
    assert y.shape == (0, 16)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(dw))


def test_layer_norm_beyond_32_bit_offsets():
    rows, dim = 2_200_000, 1000
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(5, dim, generator=gen(3), device="cuda").to(torch.bfloat16)
    x[-5:] = tail
    assert torch.equal(P.layer_norm(x)[-5:], P.layer_norm(tail))
    w = torch.ones(dim, device="cuda", requires_grad=True)
    xr = x.requires_grad_(True)
    dy = torch.zeros_like(x)
    dy[-5:] = tail.flip(0)
    dx, dw = torch.autograd.grad(P.layer_norm(xr, w), (xr, w), dy)
    t = tail.clone().requires_grad_(True)
    v = torch.ones(dim, device="cuda", requires_grad=True)
    tx, tw = torch.autograd.grad(P.layer_norm(t, v), (t, v), tail.flip(0))
    assert torch.equal(dx[-5:], tx) and not dx[:-5].any()
    within(dw, tw, 8 * U * 5 * 16, "dw")  # five terms below 16, added in two orders


# -- log-probability and entropy ----------------------------------------------------

def legal_mask(rows, n, density, seed):
    g = gen(seed)
    m = torch.rand(rows, n, generator=g, device="cuda") < density
    m[torch.arange(rows, device="cuda"), torch.randint(0, n, (rows,), generator=g, device="cuda")] = True
    if rows > 2:
        m[2] = False
    return m


def plain_logp(x, mask, a):
    """(lp, ent, p, c, logz) in 64 bits, with what the operator defines for rows and actions without a value."""
    x = x.detach().double()
    legal = torch.ones_like(x, dtype=torch.bool) if mask is None else mask.bool().expand(x.shape)
    x = torch.where(legal, x, -torch.inf)
    m = x.amax(1, keepdim=True)
    empty = m == -torch.inf
    c = x - torch.where(empty, 0, m)
    e = c.exp()
    z = torch.where(empty, 1, e.sum(1, keepdim=True))
    p, logz = e / z, z.log()
    ent = torch.where(empty, 0, logz - torch.where(e == 0, 0, p * c).sum(1, keepdim=True))
    a = a.long()[:, None]
    inside = (a >= 0) & (a < x.shape[1])
    lp = torch.where(inside, c.gather(1, a.clamp(0, x.shape[1] - 1)) - logz, 0)
    return lp[:, 0], ent[:, 0], p, c, logz


def check_logp(x, mask, a, seed=0):
    rows, n = x.shape
    x = x.detach().requires_grad_(True)
    lp, ent = P.action_log_prob(x, mask, a)
    assert lp.dtype == ent.dtype == torch.float32 and lp.shape == ent.shape == (rows,)
    with torch.no_grad():
        l2, e2 = P.action_log_prob(x, mask, a)
    within(l2, lp.detach().double(), 0, "without gradient")
    within(e2, ent.detach().double(), 0, "without gradient")
    wl, we, p, c, logz = plain_logp(x, mask, a)
    D = torch.where(torch.isfinite(c), -c, 0).amax(1).clamp(max=100)
    k = (n / 256 + 28 + D) * U
    at = torch.where(torch.isfinite(wl), wl.abs(), 0)
    within(lp, wl, 1.01 * (k + 4 * U * (at + logz[:, 0].abs())), "log_prob")
    mean = torch.where(p == 0, 0, -p * c).sum(1)
    within(ent, we, 1.01 * (2 * k * (1 + mean) + 4 * U * (logz[:, 0].abs() + mean)), "entropy")
    g = gen(seed + 5)
    u, v = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    (dx,) = torch.autograd.grad((lp, ent), x, (u, v))
    assert dx.dtype == x.dtype and dx.shape == x.shape
    inside = (a >= 0) & (a < n)
    hit = torch.zeros_like(p)
    rows_in = torch.nonzero(inside & torch.isfinite(wl))[:, 0]
    hit[rows_in, a.long()[rows_in]] = 1
    ud = u.double()[:, None] * hit.amax(1, keepdim=True)
    lgp = torch.where(p == 0, 0, c - logz)
    vd = v.double()[:, None]
    want = ud * (hit - p) - vd * torch.where(p == 0, 0, p * (lgp + we[:, None]))
    dd = torch.where(p == 0, 0, -c)
    size = p * (ud.abs() + vd.abs() * (lgp.abs() + we[:, None].abs() + 1 + mean[:, None]))
    tol = 1.01 * ((3 * k[:, None] + 2 * dd * U + 8 * U) * size + 2 * U * ud.abs() * hit)
    # where p is below the smallest normal number the kernel has 0
    within(dx, want, half_step(want, x.dtype) * 1.001 + tol + 1e-36, "dlogits")
    if mask is not None:
        assert not dx[~mask.bool().expand(x.shape)].any()
    return lp, ent, dx


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,density", [(1, 1, 1), (4, 2, 0.5), (3, 31, 0.4), (3, 32, 0.4), (5, 33, 0.2), (7, 47, 1), (9, 48, 0.1),
                                            (6, 129, 0.05), (5, 1000, 0.9), (33, 16641, 0.005), (9, 16641, 0.4),
                                            (4, 16641, 1), (4, 16648, 0.01), (3, 70001, 0.02), (2, 262144, 0.3)])
def test_action_log_prob(dtype, rows, n, density):
    x = (torch.randn(rows, n, generator=gen(rows + n), device="cuda") * 3).to(dtype)
    mask = legal_mask(rows, n, density, n)
    a = torch.where(mask, x.float() + torch.rand(rows, n, generator=gen(1), device="cuda"), -1e9).argmax(1).to(torch.int32)
    check_logp(x, mask, a)
    check_logp(x, mask.to(torch.uint8) * 7, a.long())
    check_logp(x, None, a)


@pytest.mark.parametrize("dtype", DTYPES)
def test_action_log_prob_padded_rows_and_offsets(dtype):
    """Rows that start anywhere: every phase of the mask's and the logits' vector loads."""
    for pad in range(0, 18):
        x = torch.randn(5, 200 + pad, generator=gen(pad), device="cuda").to(dtype)
        m = legal_mask(5, 200 + pad, 0.2, pad + 1)
        a = torch.randint(0, 200, (5,), generator=gen(2), device="cuda")
        check_logp(x[:, pad // 2:pad // 2 + 199], m[:, pad // 3:pad // 3 + 199], a)
        check_logp(x[:, pad // 2:pad // 2 + 199], None, a)


def test_action_log_prob_what_stands_at_masked_places_does_not_matter():
    x = torch.randn(6, 500, generator=gen(1), device="cuda")
    m = legal_mask(6, 500, 0.1, 2)
    a = m.float().argmax(1).to(torch.int32)
    ref = check_logp(x, m, a)
    for junk in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).max, torch.finfo(torch.float32).min):
        got = check_logp(torch.where(m, x, junk), m, a)
        for r, s in zip(ref, got):
            assert torch.equal(r, s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_action_log_prob_extreme_logits(dtype):
    """Legal places at -inf, at the type's lowest and highest values, all equal, and far apart."""
    big = torch.finfo(dtype).max
    x = torch.randn(8, 100, generator=gen(4), device="cuda")
    x[0, :50] = -torch.inf
    x[1] = -torch.inf
    x[2] = -big
    x[3, :] = -big
    x[3, 7] = 1.0
    x[4] = 5.0
    x[5, 10] = big
    x[6, 20:] = -big
    x[7] *= 1000
    a = torch.tensor([60, 3, 99, 7, 50, 10, 25, 0], device="cuda")
    check_logp(x.to(dtype), None, a)
    check_logp(x.to(dtype), torch.ones(100, dtype=torch.bool, device="cuda"), a)


def test_action_log_prob_nan_and_inf_at_legal_places():
    for junk in (float("nan"), float("inf")):
        x = torch.randn(5, 300, generator=gen(4), device="cuda")
        x[1, 280] = junk
        x[3] = junk
        m = torch.ones(5, 300, dtype=torch.bool, device="cuda")
        for mask in (m, None):
            xr = x.clone().requires_grad_(True)
            lp, ent = P.action_log_prob(xr, mask, torch.zeros(5, dtype=torch.int32, device="cuda"))
            assert torch.isnan(lp).tolist() == torch.isnan(ent).tolist() == [False, True, False, True, False]
            (dx,) = torch.autograd.grad(lp.sum() + ent.sum(), xr)
            assert torch.isnan(dx[1]).all() and torch.isfinite(dx[[0, 2, 4]]).all()


def test_action_log_prob_actions_without_a_value():
    """No action, out of range, illegal, at -inf, and a row without legal places."""
    x = torch.randn(7, 40, generator=gen(6), device="cuda")
    x[4, 3] = -torch.inf
    m = torch.zeros(7, 40, dtype=torch.bool, device="cuda")
    m[:, ::3] = True
    m[5:] = False
    a = torch.tensor([-1, 40, 2 ** 31 + 3, 1, 3, 0, -1], device="cuda")
    lp, ent, dx = check_logp(x, m, a)
    inf = float("inf")
    assert lp.tolist() == [0, 0, 0, -inf, -inf, -inf, 0] and ent.tolist()[5:] == [0, 0]
    xr = x.clone().requires_grad_(True)
    (d1,) = torch.autograd.grad(P.action_log_prob(xr, m, a)[0], xr, torch.ones(7, device="cuda"))
    assert not d1.any()


@pytest.mark.parametrize("kind", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_whole_numbers_of_any_type_and_none_wraps(kind):
    """2^32 + 5 is not action 5, and -2^40 not action 0, in any argument of 64 bits."""
    x = torch.randn(4, 2, 90, generator=gen(1), device="cuda")
    a = torch.tensor([5, 0, 89, 7], device="cuda")
    want = P.action_log_prob(x[:, 0], None, a)[0]
    assert torch.equal(P.action_log_prob(x[:, 0], None, a.to(kind))[0], want)
    if kind == torch.int64:
        far = torch.tensor([2 ** 32 + 5, -2 ** 40, 89, 2 ** 40 + 7], device="cuda")
        lp, _ = P.action_log_prob(x[:, 0], None, far)
        assert lp[[0, 1, 3]].tolist() == [0, 0, 0] and lp[2] == want[2]
        v = P.verify_drafts(x, far[:, None], torch.zeros(4, 1, device="cuda"), torch.zeros(4, device="cuda"),
                            lengths=torch.tensor([2 ** 32, 2 ** 32 + 1, -2 ** 33, 1], device="cuda"))
        assert v.accepted.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("op", ["norm", "logp"])
def test_second_derivatives_are_refused(op):
    x = torch.randn(3, 20, generator=gen(1), device="cuda", requires_grad=True)
    if op == "norm":
        y = P.layer_norm(x).square().sum()
    else:
        y = P.action_log_prob(x, None, torch.zeros(3, dtype=torch.int32, device="cuda"))[0].square().sum()
    (g,) = torch.autograd.grad(y, x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(g.sum(), x)


def test_results_do_not_need_gradients_where_nothing_asks_for_them():
    x = torch.randn(3, 20, device="cuda", requires_grad=True)
    a = torch.zeros(3, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        assert not P.layer_norm(x).requires_grad and not P.action_log_prob(x, None, a)[0].requires_grad
    assert not P.layer_norm(x.detach()).requires_grad
    s, lp = P.sample_actions(x, None, torch.rand(3, device="cuda"))
    assert not lp.requires_grad
    w = torch.ones(20, device="cuda", requires_grad=True)
    y = P.layer_norm(x.detach(), w)
    (gw,) = torch.autograd.grad(y.sum(), w)
    assert gw.shape == (20,)


def test_action_log_prob_one_gradient_only_and_broadcast_gradients():
    x = torch.randn(2, 5, 90, generator=gen(8), device="cuda", requires_grad=True)
    m = torch.rand(90, generator=gen(9), device="cuda") < 0.5
    m[0] = True
    a = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
    xd = x.detach().double().requires_grad_(True)
    logp = torch.log_softmax(xd.masked_fill(~m, -torch.inf), -1)
    h = -(logp.exp() * torch.where(m, logp, 0)).sum(-1)  # a gradient without 0 * inf at masked places
    tol = 200 * U * 8  # (90 / 256 + 28 + 8) u a few times over, of terms below 8
    for mine, ref in ((lambda lp, e: lp.mean(), logp[..., 0].mean()), (lambda lp, e: e.sum(), h.sum()),
                      (lambda lp, e: lp[0].sum() - 0.5 * e[:, 1].sum(), logp[0, :, 0].sum() - 0.5 * h[:, 1].sum())):
        (got,) = torch.autograd.grad(mine(*P.action_log_prob(x, m, a)), x)
        (want,) = torch.autograd.grad(ref, xd, retain_graph=True)
        within(got, want, tol, "dlogits")


def test_action_log_prob_repeated_logits():
    """One row of logits for several masks: the gradient of a broadcast input is the sum."""
    base = torch.randn(1, 64, generator=gen(3), device="cuda", requires_grad=True)
    m = legal_mask(6, 64, 0.5, 3)
    m[2, :3] = True
    a = m.float().argmax(1)
    lp, ent = P.action_log_prob(base.expand(6, 64), m, a)
    (got,) = torch.autograd.grad(lp.sum() + ent.sum(), base)
    d = base.detach().double().requires_grad_(True)
    logp = torch.log_softmax(d.expand(6, 64).masked_fill(~m, -torch.inf), 1)
    (want,) = torch.autograd.grad(logp.gather(1, a[:, None]).sum() - (logp.exp() * torch.where(m, logp, 0)).sum(), d)
    within(got, want, 6 * 200 * U * 8, "dlogits")


def test_action_log_prob_gradient_against_differences():
    """Central differences with step 2^-6: rounding 40 u of about 8 over the step, and a third derivative of about 4."""
    x = torch.randn(4, 33, generator=gen(2), device="cuda")
    m = legal_mask(4, 33, 0.6, 8)
    a = m.float().argmax(1)
    xr = x.clone().requires_grad_(True)
    lp, ent = P.action_log_prob(xr, m, a)
    (dx,) = torch.autograd.grad(lp.sum() + 0.5 * ent.sum(), xr, )
    h = 2.0 ** -6

    def f(v):
        lp, ent = P.action_log_prob(v, m, a)
        return lp.double() + 0.5 * ent.double()

    for j in range(33):
        up, dn = x.clone(), x.clone()
        up[:, j] += h
        dn[:, j] -= h
        ok = m.any(1)
        within(dx[ok, j], ((f(up) - f(dn)) / (2 * h))[ok], 40 * U * 8 / h + 4 * h * h, "dlogits")


def test_action_log_prob_backward_keeps_its_own_mask_and_actions():
    """The environment's mask and the collector's actions are overwritten before the backward pass."""
    x = torch.randn(4, 300, generator=gen(1), device="cuda", requires_grad=True)
    m = legal_mask(4, 300, 0.2, 5).to(torch.uint8)
    a = m.argmax(1).to(torch.int32)
    (want,) = torch.autograd.grad(P.action_log_prob(x, m, a)[0].sum(), x)
    lp, _ = P.action_log_prob(x, m, a)
    m.data.fill_(1)
    a.data.fill_(-1)
    (got,) = torch.autograd.grad(lp.sum(), x)
    assert torch.equal(got, want)


def test_action_log_prob_beyond_32_bit_offsets():
    rows, n = 130_000, 16641
    x = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(3, n, generator=gen(3), device="cuda").to(torch.bfloat16)
    x[-3:] = tail
    a = torch.full((rows,), 11, dtype=torch.int32, device="cuda")
    m = torch.zeros(rows, n, dtype=torch.uint8, device="cuda")
    m[:, 5::7] = 1
    m[:, 11] = 1
    for mask in (None, m):
        xr = x.requires_grad_(True)
        lp, ent = P.action_log_prob(xr, mask, a)
        (dx,) = torch.autograd.grad(lp.sum(), xr)
        t = tail.clone().requires_grad_(True)
        tl, te = P.action_log_prob(t, None if mask is None else mask[-3:], a[-3:])
        (tx,) = torch.autograd.grad(tl.sum(), t)
        # a shorter tensor's rows start at other offsets, so sums run in another order
        within(lp[-3:], tl.detach().double(), 100 * U * 4, "log_prob")
        within(ent[-3:], te.detach().double(), 400 * U * 4, "entropy")
        within(dx[-3:], tx.double(), half_step(tx.double(), torch.bfloat16) * 2 + 1e-9, "dlogits")
        del dx


# -- verification -------------------------------------------------------------------

def plain_verify(x, drafts, au, su, y, mask, lengths):
    """Game by game, in numpy and 64 bits."""
    x = x.double().cpu().numpy()
    y = None if y is None else y.double().cpu().numpy()
    games, places, n = x.shape
    mask = np.ones(x.shape, bool) if mask is None else mask.expand(games, places, n).bool().cpu().numpy()
    drafts, au, su = drafts.cpu().numpy(), au.double().cpu().numpy(), su.double().cpu().numpy()
    lens = np.full(games, places - 1) if lengths is None else np.clip(lengths.cpu().numpy(), 0, places - 1)
    acc, out, lps = np.zeros(games, int), np.full((games, places), -1), np.zeros((games, places))

    def dist(row, legal):
        row = np.where(legal, row, -np.inf)
        if not (row > -np.inf).any():
            return None if not np.isnan(row).any() else np.nan, row
        if np.isnan(row).any() or (row == np.inf).any():
            return np.nan, row
        c = row - row.max()
        e = np.exp(c)
        return e / e.sum(), c - np.log(e.sum())

    for gm in range(games):
        for i in range(places):
            legal = mask[gm, i]
            p, lp = dist(x[gm, i], legal)
            q, a = None, -1
            if i < lens[gm]:
                a = int(drafts[gm, i])
                q = dist(y[gm, i], legal)[0] if y is not None else (np.arange(n) == a).astype(float) if 0 <= a < n else None
            broken = np.isscalar(p) or np.isscalar(q)
            if i < lens[gm] and 0 <= a < n and legal[a] and p is not None and not broken:
                if au[gm, i] * (0.0 if q is None else q[a]) < p[a]:
                    out[gm, i], lps[gm, i] = a, lp[a]
                    continue
            acc[gm] = i
            if broken:
                lps[gm, i] = np.nan
            elif p is not None:
                w = p
                if q is not None and np.maximum(p - q, 0).sum() > 2.0 ** -40:
                    w = np.maximum(p - q, 0)
                run = np.cumsum(w)
                over = np.nonzero(run > (su[gm] if su[gm] > 0 else 0.0) * run[-1])[0]
                out[gm, i] = over[0] if len(over) else np.nonzero(w > 0)[0][-1]
                lps[gm, i] = lp[out[gm, i]]
            break
    return acc, out, lps


def check_verify(x, drafts, au, su, y=None, mask=None, lengths=None):
    v = P.verify_drafts(x, drafts, au, su, draft_logits=y, mask=mask, lengths=lengths)
    acc, out, lps = plain_verify(x, drafts, au, su, y, mask, lengths)
    assert v.accepted.dtype == v.actions.dtype == torch.int32 and v.log_probs.dtype == torch.float32
    assert np.array_equal(v.accepted.cpu().numpy(), acc)
    assert np.array_equal(v.actions.cpu().numpy(), out)
    # 64-bit values, rounded once: half a step of 32 bits, and 2^-40 for the orders of the sums
    w = torch.from_numpy(lps).cuda()
    tol = w.abs().nan_to_num() * U * 1.001 + 2.0 ** -40
    if mask is None:
        # a kept draft's log Z comes from a 32-bit sum.  These calls have at most 64 games, so a cluster has eight CTAs or
        # at most 1,024 places for each, and a lane at most max(n / 256, 32) terms: each added once (u) and with an
        # exponential of 4 u (2^-22) after three roundings of its argument (its size, weighted by the probabilities, is at
        # most log2 n = 18: 3 * 18 u), 4 u for each of at most n / 1024 + 2 times that the maximum rises, and five joins of
        # 5 u, in all below (2 max(n / 256, 32) + 150) u
        assert x.shape[0] <= 64
        kept = torch.arange(out.shape[1], device="cuda")[None, :] < torch.from_numpy(acc).cuda()[:, None]
        tol = tol + kept * ((2 * max(x.shape[2] / 256, 32) + 150) * U)
    within(v.log_probs, w, tol, "log_probs")
    return v


def drafted(games, d, n, dtype, seed, density=None, noise=0.5):
    g = gen(seed)
    x = torch.randn(games, d + 1, n, generator=g, device="cuda") * 2
    y = (x[:, :d] + noise * torch.randn(games, d, n, generator=g, device="cuda")).to(dtype)
    mask = None
    if density is not None:
        mask = torch.rand(games, d + 1, n, generator=g, device="cuda") < density
        mask[torch.rand(games, d + 1, generator=g, device="cuda") < 0.05] = False
    gum = -torch.log(-torch.log(torch.rand(y.shape, generator=g, device="cuda").clamp(1e-9, 1 - 1e-6)))
    s = y.float() + gum
    if mask is not None:
        s = s.masked_fill(~mask[:, :d], -torch.inf)
    a = s.argmax(-1) if d else torch.zeros(games, 0, dtype=torch.int64, device="cuda")
    return (x.to(dtype), a.to(torch.int32), torch.rand(games, d, generator=g, device="cuda"),
            torch.rand(games, generator=g, device="cuda"), y, mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("games,d,n,density", [(1, 0, 1, None), (3, 0, 40, 0.3), (4, 1, 2, None), (9, 3, 31, 0.5), (9, 3, 33, 0.5),
                                               (40, 5, 129, 0.2), (30, 4, 1000, None), (64, 4, 16641, 0.005),
                                               (20, 8, 16641, 0.3), (12, 2, 16641, None), (5, 17, 300, 0.1),
                                               (2, 1, 262144, 0.01), (2, 1, 262144, None)])
def test_verify_drafts(dtype, games, d, n, density):
    x, a, au, su, y, mask = drafted(games, d, n, dtype, games + n, density)
    check_verify(x, a, au, su, y if d else None, mask)
    check_verify(x, a.long(), au, su, None, mask)
    ln = torch.randint(0, d + 1, (games,), generator=gen(3), device="cuda")
    check_verify(x, a, au, su, y if d else None, None if mask is None else mask.to(torch.uint8) * 200, ln)
    check_verify(x, a, au, su, None, mask, ln.to(torch.int32))


@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("layout", ["spread", "first", "last", "steps"])
@pytest.mark.parametrize("d", [0, 3])
def test_verify_drafts_longer_than_the_list(d, layout, scored):
    """More legal actions than a warp's list holds (320), so that it takes them in parts: one more, exactly two and three
    lists, parts that end inside a word of the mask, all actions; the points of the draw at both ends and in between."""
    n = 5003
    counts = [0, 1, 319, 320, 321, 345, 352, 639, 640, 641, 960, 961, 1500, n - 1, n]
    games = 3 * len(counts)
    x, _, au, su, y, _ = drafted(games, d, n, torch.float32, 40 + d, noise=0.7)
    g = gen(50)
    mask = torch.zeros(games, d + 1, n, dtype=torch.bool, device="cuda")
    for k in range(games):
        c = counts[k % len(counts)]
        at = {"spread": torch.randperm(n, generator=g, device="cuda")[:c], "first": torch.arange(c, device="cuda"),
              "last": torch.arange(n - c, n, device="cuda"),
              "steps": torch.arange(c, device="cuda") * max(1, n // max(1, c))}[layout]
        mask[k, :, at] = True
    a = torch.where(mask[:, :d], y + x[:, :d], -torch.inf).argmax(-1).to(torch.int32)
    su[:len(counts)], su[len(counts):2 * len(counts)] = 0, 1 - 2 ** -24
    check_verify(x, a, au, su, y if d and scored else None, mask)
    # NaN, +inf, rows of -inf and -inf but for the last part, in legal places behind the first list
    last = n - 1 - mask.flip(-1).float().argmax(-1)
    for k, v in ((4, float("nan")), (5, float("inf")), (12, float("-inf"))):
        x[k, 0, last[k, 0]] = v
    x[13] = -torch.inf
    x[14, :, :n - 40] = -torch.inf
    if d:
        y[28, :, :n - 40] = -torch.inf
        y[27, 0, last[27, 0]] = float("nan")
    check_verify(x, a, au, su, y if d and scored else None, mask)


def test_verify_drafts_of_the_target_itself_keeps_everything():
    x, a, au, su, y, mask = drafted(50, 6, 500, torch.float32, 1, 0.3, noise=0.0)
    mask[..., 0] = True
    a = torch.where((a == 0) | ~mask[:, :6].any(-1), 0, a)
    v = check_verify(x, a, au, su, y, mask)
    assert (v.accepted == 6).all()


def test_verify_drafts_bad_drafts_and_lengths():
    """-1, out of range, illegal and impossible drafts, lengths outside [0, D]."""
    x, a, au, su, y, mask = drafted(24, 3, 90, torch.float32, 2, 0.4)
    a[0, 0], a[1, 0], a[2, 1], a[3, 0] = -1, 90, 2 ** 31 - 1, -2 ** 31
    for gm in range(4, 12):
        a[gm, 0] = (~mask[gm, 0]).float().argmax()
    y[12:16] = -torch.inf        # the draft could not have played at all
    y[16:20, :, ::2] = -torch.inf
    x[20, 1] = -torch.inf
    ln = torch.tensor([-5, 99] * 12, dtype=torch.int32, device="cuda")
    for lengths in (None, ln):
        check_verify(x, a, au, su, y, mask, lengths)
        check_verify(x, a, au, su, None, mask, lengths)


@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("n", [50, 16641])
@pytest.mark.parametrize("scored", [True, False])
def test_verify_drafts_at_the_borders(masked, n, scored):
    """accept_u at p / q itself and the 32-bit numbers next to it (at most 2^-24 away, relatively), and sample_u next
    to a border between two actions: the choices are those of 64 bits."""
    games, d = 60, 3
    x, a, au, su, y, mask = drafted(games, d, n, torch.float32, 11 + n, 0.2 if masked else None)
    legal = torch.ones(x.shape, dtype=torch.bool, device="cuda") if mask is None else mask

    def dist(t, m):
        t = t.double().masked_fill(~m, -torch.inf)
        return (t - t.amax(-1, keepdim=True).clamp(min=-1e9)).softmax(-1).nan_to_num()

    p, q = dist(x, legal), dist(y, legal[:, :d])
    at = a.long().clamp(min=0)[..., None]
    ratio = p[:, :d].gather(2, at)[..., 0] / (q.gather(2, at)[..., 0] if scored else 1.0)
    border = ratio.clamp(max=1 - 2.0 ** -24).nan_to_num().float()
    step = torch.arange(games, device="cuda")[:, None] % 3 - 1
    au = torch.where(step == 0, border, torch.nextafter(border, step.float().expand(games, d) * 10)).clamp(0, 1 - 2.0 ** -24)
    w = p[:, d]
    run = w.cumsum(1)
    j = torch.multinomial(w + 1e-12, 1, generator=gen(4))
    su = run.gather(1, j)[:, 0].clamp(max=1 - 2.0 ** -24).float()
    for lengths in (None, torch.zeros(games, dtype=torch.int32, device="cuda")):
        v = P.verify_drafts(x, a, au, su, draft_logits=y if scored else None, mask=mask, lengths=lengths)
        acc, out, _ = plain_verify(x, a, au, su, y if scored else None, mask, lengths)
        assert np.array_equal(v.accepted.cpu().numpy(), acc) and np.array_equal(v.actions.cpu().numpy(), out)


def test_verify_drafts_extreme_random_numbers():
    """0, the largest number below 1, and, though not allowed, 1 and more, negative ones and NaN."""
    x, a, au, su, y, mask = drafted(40, 3, 200, torch.float32, 5, 0.2)
    su[:8] = 0
    su[8:16] = 1 - 2.0 ** -24
    su[16:20], su[20:22], su[22:24] = 1.0, 7.5, -2.0
    su[24:27] = float("nan")
    su[27:30] = float("inf")
    au[::3] = 0
    au[1::3] = 1 - 2.0 ** -24
    for y_ in (y, None):
        v = P.verify_drafts(x, a, au, su, draft_logits=y_, mask=mask)
        s2 = torch.where(torch.isinf(su), 9.0, su)
        acc, out, _ = plain_verify(x, a, au, s2, y_, mask, None)
        assert np.array_equal(v.accepted.cpu().numpy(), acc) and np.array_equal(v.actions.cpu().numpy(), out)


def test_verify_drafts_nan_and_inf():
    x, a, au, su, y, mask = drafted(30, 3, 64, torch.float32, 6, 0.5)
    x[0, 0], x[1, 1], y[2, 0], y[3, 1] = float("nan"), float("inf"), float("nan"), float("inf")
    x[4] = torch.where(mask[4], x[4], float("nan"))   # only at masked places: not looked at
    y[5] = torch.where(mask[5, :3], y[5], float("inf"))
    check_verify(x, a, au, su, y, mask)
    check_verify(x, a, au, su, None, mask)
    check_verify(x, a, au, su, y, None)


def test_verify_drafts_strides():
    """Interleaved games, sliced places and actions, one mask for all, repeated logits."""
    x, a, au, su, y, mask = drafted(10, 4, 211, torch.float32, 8, 0.3)
    wide = torch.zeros(5, 10, 230, device="cuda")
    wide[:, :, 7:218] = x.transpose(0, 1)
    wm = torch.zeros(5, 10, 301, dtype=torch.uint8, device="cuda")
    wm[:, :, 33:244] = mask.transpose(0, 1)
    check_verify(wide[:, :, 7:218].transpose(0, 1), a.t().contiguous().t(), au, su, y.transpose(1, 2).contiguous().transpose(1, 2),
                 wm[:, :, 33:244].transpose(0, 1))
    check_verify(x, a, au, su, y, mask[:1, :1])
    check_verify(x[:1].expand(10, 5, 211), a, au, su, y, mask[0, 0])


def test_sample_actions_shapes_and_empty():
    x = torch.randn(3, 4, 70, generator=gen(1), device="cuda")
    m = legal_mask(12, 70, 0.2, 4).view(3, 4, 70)
    u = torch.rand(3, 4, generator=gen(2), device="cuda")
    a, lp = P.sample_actions(x, m, u)
    v = check_verify(x.view(12, 1, 70), torch.zeros(12, 0, dtype=torch.int32, device="cuda"),
                     torch.zeros(12, 0, device="cuda"), u.view(12), None, m.view(12, 1, 70))
    assert torch.equal(a.view(12, 1), v.actions) and torch.equal(lp.view(12, 1), v.log_probs)
    assert int(a[0, 2]) == -1 and float(lp[0, 2]) == 0
    one, _ = P.sample_actions(x[0, 0], m[0, 0], u[0, 0])
    assert one.shape == () and one == a[0, 0]
    a, lp = P.sample_actions(x[:0], m[:0], u[:0])
    assert a.shape == lp.shape == (0, 4)
    xr = torch.zeros(0, 9, device="cuda", requires_grad=True)
    lp, ent = P.action_log_prob(xr, None, torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert torch.autograd.grad(lp.sum() + ent.sum(), xr)[0].shape == (0, 9)


def test_samples_follow_the_probabilities():
    """2^16 evenly spread points: an action's share is its probability to one point either way (and the 2^-24
    steps of the points)."""
    n = 2 ** 16
    x = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.1], device="cuda")
    m = torch.tensor([1, 1, 0, 1, 1], dtype=torch.uint8, device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    a, lp = P.sample_actions(x.expand(n, 5), m, u)
    share = torch.bincount(a.long(), minlength=5).double() / n
    p = torch.where(m != 0, x.double(), -torch.inf).softmax(0)
    assert ((share - p).abs() <= 1.01 / n).all()


def test_verified_play_is_distributed_as_the_target():
    """Over a grid of (draft, accept_u, sample_u) the first action's share is the target's probability: the
    draft's own probability as weight, 256 x 256 points each; borders cost two points in 256 either way."""
    k = 256
    x = torch.tensor([0.2, 1.4, -0.7, 0.9], device="cuda")
    y = torch.tensor([1.0, 0.1, 0.3, -1.2], device="cuda")
    p, q = x.double().softmax(0), y.double().softmax(0)
    u = (torch.arange(k, device="cuda") + 0.5) / k
    au, su = u.repeat_interleave(k), u.repeat(k)
    share = torch.zeros(4, dtype=torch.float64, device="cuda")
    for d in range(4):
        v = P.verify_drafts(x.expand(k * k, 2, 4), torch.full((k * k, 1), d, device="cuda"), au[:, None], su,
                            draft_logits=y.expand(k * k, 1, 4))
        share += q[d] * torch.bincount(v.actions[:, 0].long(), minlength=4) / (k * k)
    assert ((share - p).abs() <= 4 / k).all(), (share, p)


def test_verify_drafts_beyond_32_bit_offsets():
    games, d, n = 33_000, 3, 16641
    x, a, au, su, y, mask = drafted(6, d, n, torch.bfloat16, 3, 0.01)
    big = torch.zeros(games, d + 1, n, dtype=torch.bfloat16, device="cuda")
    big[-6:] = x
    legal = torch.zeros(games, d + 1, n, dtype=torch.uint8, device="cuda")
    legal[-6:] = mask
    drafts = torch.zeros(games, d, dtype=torch.int32, device="cuda")
    drafts[-6:] = a
    u, r = torch.full((games, d), 0.5, device="cuda"), torch.full((games,), 0.5, device="cuda")
    u[-6:], r[-6:] = au, su
    for m in (legal, None):
        v = P.verify_drafts(big, drafts, u, r, mask=m)
        w = check_verify(x, a, au, su, None, None if m is None else mask)
        assert torch.equal(v.accepted[-6:], w.accepted) and torch.equal(v.actions[-6:], w.actions)
        if m is not None:  # nothing legal anywhere else
            assert not v.accepted[:-6].any() and (v.actions[:-6] == -1).all() and not v.log_probs[:-6].any()


# -- streams and graphs ------------------------------------------------------------------

def test_other_streams():
    """Work on a side stream, on tensors made on the default one."""
    x = torch.randn(200, 700, generator=gen(1), device="cuda", requires_grad=True)
    m = legal_mask(200, 700, 0.1, 2)
    u = torch.rand(200, generator=gen(3), device="cuda")

    def work():
        y = P.layer_norm(x)
        a, _ = P.sample_actions(y, m, u)
        lp, ent = P.action_log_prob(y, m, a)
        return a, lp.detach(), torch.autograd.grad(lp.sum() + ent.sum(), x)[0]

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = work()
    torch.cuda.current_stream().wait_stream(side)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_two_threads_at_once():
    """Calls of two threads, each on a stream of its own, forward and backward."""
    import threading
    x = torch.randn(200, 700, generator=gen(1), device="cuda")
    m = legal_mask(200, 700, 0.1, 2)
    u = torch.rand(200, generator=gen(3), device="cuda")

    def work():
        leaf = x.clone().requires_grad_(True)
        y = P.layer_norm(leaf)
        a, _ = P.sample_actions(y, m, u)
        lp, ent = P.action_log_prob(y, m, a)
        return a, lp.detach(), torch.autograd.grad(lp.sum() + ent.sum(), leaf)[0]

    want = work()
    torch.cuda.synchronize()
    wrong = []

    def run():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = work()
                torch.cuda.current_stream().synchronize()
                wrong.extend(1 for g, w in zip(got, want) if not torch.equal(g, w))

    threads = [threading.Thread(target=run) for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


def test_graphs_replay_on_new_inputs():
    """Two captured training steps share nothing: replayed in turn and on two streams at once, each gives what an
    eager step gives on the same inputs."""
    def make(seed):
        g = gen(seed)
        return (torch.randn(300, 128, generator=g, device="cuda"), legal_mask(300, 128, 0.2, seed),
                torch.rand(300, generator=g, device="cuda"))

    def step(x, w, m, u):
        y = P.layer_norm(x, w)
        a, _ = P.sample_actions(y, m, u)
        lp, ent = P.action_log_prob(y, m, a)
        return (a, lp.detach(), *torch.autograd.grad(lp.sum() - 0.1 * ent.sum(), (x, w)))

    graphs = []
    for s in (1, 2):
        x, m, u = make(s)
        x.requires_grad_(True)
        w = torch.ones(128, device="cuda", requires_grad=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, w, m, u)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(x, w, m, u)
        graphs.append((gr, x, w, m, u, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rnd in range(3):
        for k, (gr, x, w, m, u, out) in enumerate(graphs):
            nx, nm, nu = make(10 * rnd + k + 3)
            with torch.no_grad():
                x.copy_(nx)
            m.copy_(nm)
            u.copy_(nu)
        torch.cuda.synchronize()
        for st, (gr, *_) in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for gr, x, w, m, u, out in graphs:
            for o, e in zip(out, step(x, w, m, u)):
                assert torch.equal(o, e)
