"""linear_cross_entropy where rows of its operands differ by many powers of ten, and where
its packed kernels (more than 128 tokens over more than 128 rows of vocabulary) are what
runs. The definition is computed in float64.

Bounds. A packed float32 operand keeps 22 bits of an element (2^-22, with the dropped
product of two low parts) down to 2^-39 of its row's largest, and sums are float32 (about
2^-24 a term's magnitude, few hundred terms in random signs): with a = the row maxima of h
and b those of W, a logit is off by at most

    e_z = 2^-20 Σ|h w| + 2^-38 (a Σ|w| + b Σ|h|).

p = exp(z - lse) is off by p (exp(2 max e_z + 2e-6) - 1). A product C = A·B whose K runs
over B's packed rows of largest magnitude β, where A was scaled by its rows' largest terms,
is off by 2^-20 Σ|A||B| + 2^-37 (Σ|A|β + K max|A|β). Where the kernels use float32
instructions (few tokens, a small vocabulary) the same bounds hold with room.
"""

from __future__ import annotations

import math

import pytest
import torch

import sparsecore_amd as slk

pytestmark = pytest.mark.gpu

U20, U37, U38 = 2.0 ** -20, 2.0 ** -37, 2.0 ** -38


def product(a, b, ea):
    """a·b and its bound, a off by ea."""
    c = a @ b
    beta = b.abs().amax(1)
    terms = a.abs() @ beta
    most = (a.abs() * beta).amax(1)
    err = ea @ b.abs() + U20 * (a.abs() @ b.abs()) \
        + (U37 * (terms + b.shape[0] * most))[:, None]
    return c, err


def reference(h, w, t, up):
    """(losses, dh, dw) as (value, bound) pairs, for upstream gradients of each token."""
    h, w, up = h.detach().double(), w.detach().double(), up.double()
    live = t != -100
    h = torch.where(live[:, None], h, 0.0)
    hit = (t[:, None] == torch.arange(w.shape[0], device=t.device)).double()
    z = h @ w.t()
    ez = U20 * (h.abs() @ w.abs().t()) + U38 * (
        h.abs().amax(1)[:, None] * w.abs().sum(1) + w.abs().amax(1) * h.abs().sum(1)[:, None])
    e = 2 * ez.amax(1, keepdim=True) + 2e-6
    lse = torch.logsumexp(z, 1, keepdim=True)
    losses = torch.where(live, lse.squeeze(1) - (z * hit).sum(1), 0.0)
    loss_err = torch.where(live, e.squeeze(1) + 2e-6 * (1 + lse.squeeze(1).abs()
                                                      + (z * hit).sum(1).abs()), 0.0)
    p = torch.exp(z - lse)
    ep = p * torch.expm1(e.clamp(max=80.0)) + 2.0 ** -126
    g = torch.where(live, up, 0.0)[:, None]
    # target's p - 1 rounds at 2^-24 of 1 where p is near 1
    dl, edl = (p - hit) * g, (ep + 2.0 ** -24 * hit) * g.abs()
    dh, dw = product(dl, w, edl), product(dl.t(), h, edl.t())
    return (losses, loss_err), dh, dw


def within(got, pair, what):
    want, err = pair
    far = (got.detach().double() - want).abs() - err
    assert bool((far <= 0).all()), f"{what}: {int((far > 0).sum())} beyond, by {float(far.max()):.3g}"


def inputs(n, d, v, dev, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, d, generator=g).to(dtype).to(dev)
    w = (torch.randn(v, d, generator=g) * 2 / math.sqrt(d)).to(dtype).to(dev)
    return h, w, torch.randint(0, v, (n,), generator=g).to(dev)


def check(h, w, t, up=None, reduction="none"):
    n = t.numel()
    up = torch.ones(n, device=h.device) if up is None else up
    h, w = h.clone().requires_grad_(), w.clone().requires_grad_()
    losses, dh, dw = reference(h, w, t, up)
    loss = slk.linear_cross_entropy(h, w, t, reduction="none")
    within(loss, losses, "loss")
    gh, gw = torch.autograd.grad(loss, [h, w], up)
    within(gh, dh, "dh")
    within(gw, dw, "dw")


def mixed(n, low, high, dev, seed):
    """n powers of ten between 10^low and 10^high, in no order."""
    s = torch.logspace(low, high, n, dtype=torch.float64)
    return s[torch.randperm(n, generator=torch.Generator().manual_seed(seed))].float().to(dev)


SIZES = [(40, 64, 300), (300, 64, 520), (700, 130, 1500), (300, 64, 65)]


@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("low,high", [(-6, 0), (-6, 6), (-12, 0)])
def test_hidden_states_of_any_magnitude(dev, n, d, v, low, high):
    h, w, t = inputs(n, d, v, dev, 1)
    check(h * mixed(n, low, high, dev, 1)[:, None], w, t)


@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("low,high", [(-6, 0), (-12, 0), (-8, 4)])
def test_rows_of_the_head_of_any_magnitude(dev, n, d, v, low, high):
    h, w, t = inputs(n, d, v, dev, 2)
    check(h, w * mixed(v, low, high, dev, 2)[:, None], t)


@pytest.mark.parametrize("n,d,v", SIZES)
def test_upstream_gradients_of_any_magnitude(dev, n, d, v):
    h, w, t = inputs(n, d, v, dev, 3)
    check(h, w, t, mixed(n, -12, 0, dev, 3))
    check(h, w, t, mixed(n, -30, 6, dev, 4))
    check(h * mixed(n, -4, 0, dev, 5)[:, None], w * mixed(v, -6, 0, dev, 6)[:, None], t,
          mixed(n, -6, 6, dev, 7))


@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("big", [1e5, 1e8, 1e12])
def test_one_large_token_leaves_the_others_alone(dev, n, d, v, big):
    """One element of one token, as models have in their first tokens, and one of a row
    of the head."""
    h, w, t = inputs(n, d, v, dev, 4)
    h[7, 3] = big
    check(h, w, t)
    h, w, t = inputs(n, d, v, dev, 5)
    w[v // 2, 1] = big
    h[:, 1] = h[:, 1].abs() * -1.0  # the row's logits are far below the others'
    check(h, w, t)


@pytest.mark.parametrize("n,d,v", SIZES)
def test_rows_that_softmax_hardly_reaches(dev, n, d, v):
    """Half of the vocabulary with probabilities near 1e-12 and no token's target: the
    gradient of its rows is that small, and as exact as the others'."""
    h, w, t = inputs(n, d, v, dev, 6)
    h[:, 0] = 1.0
    w[:, 0] = 0.0
    w[v // 2:, 0] = -24.0
    t %= v // 2
    check(h, w, t)
    gw, = torch.autograd.grad(slk.linear_cross_entropy(h, w.requires_grad_(), t), w)
    assert bool((gw[v // 2:, 1:] != 0).any(1).all())


def test_pieces_keep_their_own_scales(dev):
    """More logits than a piece of the backward holds, rows of the head from 1e-9 to 1:
    dh adds pieces that were scaled differently."""
    n, d, v = 4200, 40, 70000
    h, w, t = inputs(n, d, v, dev, 7)
    w *= torch.logspace(-9, 0, v, device=dev)[:, None]
    up = mixed(n, -6, 0, dev, 8)
    h, w = h.requires_grad_(), w.requires_grad_()
    gh, gw = torch.autograd.grad(slk.linear_cross_entropy(h, w, t, reduction="none"), [h, w], up)
    some = torch.arange(0, n, 97, device=dev)
    _, dh, _ = reference(h[some], w, t[some], up[some])
    within(gh[some], dh, "dh")
    # rows of dw need all tokens' softmax: lse once, then a block of rows at a time
    hd, wd = h.detach().double(), w.detach().double()
    lse = torch.cat([torch.logsumexp(x @ wd.t(), 1) for x in hd.split(300)])[:, None]
    for lo in range(0, v, 7000):
        rows = slice(lo, lo + 7000)
        z = hd @ wd[rows].t()
        p = torch.exp(z - lse)
        hit = (t[:, None] == torch.arange(v, device=dev)[rows]).double()
        dl = (p - hit) * up.double()[:, None]
        edl = (p * 1e-4 + 2.0 ** -24 * hit) * up.double()[:, None]  # |z| below 10: e_z below 2e-5
        within(gw[rows], product(dl.t(), hd, edl.t()), f"dw from {lo}")


@pytest.mark.parametrize("n,d,v", SIZES)
def test_extreme_magnitudes_stay_finite(dev, n, d, v):
    """Tiny rows of one operand against huge ones of the other: no power of two in
    between overflows or is lost."""
    h, w, t = inputs(n, d, v, dev, 9)
    check(h * 1e30, w * 1e-30, t)
    check(h * 1e-30, w * 1e30, t)
    check(h * 1e-36, w * 1e-3, t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", [(8, 64, 300), (40, 64, 300), (100, 64, 300), (300, 64, 520),
                                   (700, 130, 1500), (300, 64, 65), (9000, 40, 65)])
@pytest.mark.parametrize("power", [10, 30, 60, 110])
def test_logits_of_any_size(dev, dtype, n, d, v, power):
    """Whole numbers times 2^power: every product and sum is exact and the softmax is 0
    but at the largest logits, which share it. One rounding of each result, of dl before it
    (2^-8 in bfloat16), of the losses' difference and logarithm."""
    g = torch.Generator().manual_seed(n + power)
    h = torch.randint(-2, 3, (n, d), generator=g).double()
    w = torch.randint(-2, 3, (v, d), generator=g).double()
    t = torch.randint(0, v, (n,), generator=g)
    z = h @ w.t()
    top = z.amax(1, keepdim=True)
    p = (z == top).double()
    ties = p.sum(1, keepdim=True)
    p /= ties
    rest = (top - z.gather(1, t[:, None])).squeeze(1)
    rest = torch.ldexp(rest, torch.tensor(power)) + ties.squeeze(1).log()
    dl = p.scatter_add(1, t[:, None], -torch.ones(n, 1, dtype=torch.float64))
    half = power // 2
    hs, ws = torch.ldexp(h, torch.tensor(half)), torch.ldexp(w, torch.tensor(power - half))
    hg = hs.to(dtype).to(dev).requires_grad_()
    wg = ws.to(dtype).to(dev).requires_grad_()
    loss = slk.linear_cross_entropy(hg, wg, t.to(dev), reduction="none")
    assert bool(((loss.double().cpu() - rest).abs() <= 1e-6 * rest.abs() + 1e-6).all())
    gh, gw = torch.autograd.grad(loss, [hg, wg], torch.ones(n, device=dev))
    u = 2.0 ** -7 if dtype is torch.bfloat16 else 2.0 ** -19
    for got, a, b in ((gh, dl, ws), (gw, dl.t(), hs)):
        err = (got.double().cpu() - a @ b).abs() - u * (a.abs() @ b.abs())
        assert bool((err <= 0).all()), float(err.max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", [(2100, 40, 60000), (700, 130, 1500)])
def test_the_backwards_logits_are_the_forwards(dev, dtype, n, d, v):
    """Logits near 1e6, whose last bit is 0.06: where the largest stands 40 above the
    others the softmax is 1 there, to the last bit if both passes sum in the same order,
    and dh = W[largest] - W[target] (in the first size a piece of the backward has other
    tiles than the whole vocabulary)."""
    h, w, t = inputs(n, d, v, dev, 10, dtype)
    w = (w.double() / w.double().norm(dim=1, keepdim=True)).to(dtype)  # the largest: by angle
    h = (h.double() * (1e6 / h.double().norm(dim=1, keepdim=True))).to(dtype)
    top = torch.empty(n, dtype=torch.int64, device=dev)
    alone = torch.empty(n, dtype=torch.bool, device=dev)
    for i in range(0, n, 300):
        z, at = (h[i:i + 300].double() @ w.double().t()).topk(2, dim=1)
        top[i:i + 300], alone[i:i + 300] = at[:, 0], z[:, 0] - z[:, 1] > 40
    assert int(alone.sum()) > n // 2
    h.requires_grad_()
    loss = slk.linear_cross_entropy(h, w, t, reduction="none")
    gh, = torch.autograd.grad(loss, h, torch.ones(n, device=dev))
    want = w.double()[top] - w.double()[t]
    u = 2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -19
    err = (gh.double() - want).abs() - u * (w.double()[top].abs() + w.double()[t].abs())
    assert bool((err[alone] <= 0).all()), float(err[alone].max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", [(20, 64, 300), (40, 64, 300), (300, 64, 520), (300, 64, 65)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_one_tokens_upstream_gradient_reaches_its_own_dh_alone(dev, dtype, n, d, v, bad):
    h, w, t = inputs(n, d, v, dev, 11, dtype)
    t[4] = -100
    h.requires_grad_()
    loss = slk.linear_cross_entropy(h, w, t, reduction="none")
    up = torch.randn(n, generator=torch.Generator().manual_seed(12)).to(dev)
    clean, = torch.autograd.grad(loss, h, up, retain_graph=True)
    up[7] = bad
    up[4] = bad  # ignored: reaches nothing
    got, = torch.autograd.grad(loss, h, up)
    keep = torch.arange(n, device=dev) != 7
    assert torch.equal(got[keep], clean[keep])
    assert not bool(torch.isfinite(got[7]).any()) and bool((got[4] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [20, 300])
def test_upstream_gradients_that_are_all_zero(dev, dtype, n):
    h, w, t = inputs(n, 64, 300, dev, 13, dtype)
    h.requires_grad_(), w.requires_grad_()
    loss = slk.linear_cross_entropy(h, w, t, reduction="none")
    gh, gw = torch.autograd.grad(loss, [h, w], torch.zeros(n, device=dev))
    assert bool((gh == 0).all()) and bool((gw == 0).all())
