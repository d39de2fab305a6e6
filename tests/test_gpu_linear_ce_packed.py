"""linear_cross_entropy's packed kernels: what its other tests check at sizes that the ways
for few tokens and small vocabularies take, here with more than 128 tokens over more than
128 rows."""

from __future__ import annotations

import math

import pytest
import torch

import sparsecore_amd as slk
from test_gpu_linear_ce import make, reference, within

pytestmark = pytest.mark.gpu

SIZES = [(200, 64, 300), (700, 130, 1030)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
def test_ignored_tokens_reach_nothing(dev, dtype, n, d, v, bad):
    h, w, t = make(n, d, v, dtype, dev, 1)
    out = (torch.arange(n, device=dev) % 3 == 0)[:, None]
    t[::3] = -100
    runs = []
    for x in (torch.where(out, bad, h), torch.where(out, 0, h)):
        x, y = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = slk.linear_cross_entropy(x, y, t)
        runs.append((loss.detach(), *torch.autograd.grad(loss, [x, y])))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert bool((runs[0][1][::3] == 0).all()) and bool(torch.isfinite(runs[0][2]).all())
    live = int((t != -100).sum())
    up = torch.full((n,), 1.0 / live, dtype=torch.float64, device=dev)
    losses, lerr, dh, eh, dw, ew = reference(h, w, t, up)
    within(runs[0][0], losses.sum() / live, lerr.sum() / live + 1e-6, "loss")
    within(runs[0][1], dh, eh + 2e-7 * dh.abs(), "dh")
    within(runs[0][2], dw, ew + 2e-7 * dw.abs(), "dw")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", SIZES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_live_non_finite_value_stays_in_its_loss_and_dh(dev, dtype, n, d, v, bad):
    h, w, t = make(n, d, v, dtype, dev, 2)
    x = h.clone().requires_grad_()
    clean = slk.linear_cross_entropy(x, w, t, reduction="none")
    dclean, = torch.autograd.grad(clean, x, torch.ones_like(clean))
    h[7, 3] = bad
    h.requires_grad_()
    got = slk.linear_cross_entropy(h, w, t, reduction="none")
    keep = torch.arange(n, device=dev) != 7
    assert torch.equal(got[keep], clean[keep]) and not bool(torch.isfinite(got[7]))
    gh, = torch.autograd.grad(got, h, torch.ones_like(got))
    assert torch.equal(gh[keep], dclean[keep]) and bool(torch.isnan(gh[7]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_targets_outside_the_vocabulary(dev, dtype, n, d, v):
    """Their loss is NaN and their gradient the softmax's; the others keep theirs."""
    h, w, t = make(n, d, v, dtype, dev, 3)
    clean = slk.linear_cross_entropy(h, w, t, reduction="none")
    t[2], t[5], t[n - 1] = v, -7, 1 << 40
    out = [2, 5, n - 1]
    keep = [i for i in range(n) if i not in out]
    h.requires_grad_(), w.requires_grad_()
    got = slk.linear_cross_entropy(h, w, t, reduction="none")
    assert bool(torch.isnan(got[out]).all()) and torch.equal(got[keep], clean[keep])
    gh, gw = torch.autograd.grad(got, [h, w], torch.ones(n, device=dev))
    assert bool(torch.isfinite(gw).all())
    z = h.detach().double() @ w.detach().double().t()
    want = torch.softmax(z[out], 1) @ w.detach().double()
    # dl to 2^-8 in bfloat16 (p to 1e-4 otherwise: |z| is below 30), then the result
    u = 2.0 ** -7 if dtype is torch.bfloat16 else 1e-4
    terms = torch.softmax(z[out], 1) @ w.detach().double().abs()
    assert bool(((gh[out].double() - want).abs() <= u * terms).all())


@pytest.mark.parametrize("n,d,v", SIZES)
def test_gradient_against_differences(dev, n, d, v):
    """Central differences along random directions of length 1, step 2^-6: truncation is
    step² times a third derivative of order 1 / n at most (of a mean of losses whose logits
    move by at most |h| or |w|, about 8 and 2, cubed: 3e-3 · 512 / n), rounding about
    2^-20 / step."""
    h, w, t = make(n, d, v, torch.float32, dev, 4)
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    grads = torch.autograd.grad(slk.linear_cross_entropy(hg, wg, t), [hg, wg])
    step = 2.0 ** -6
    for k, g in enumerate(grads):
        way = torch.randn(g.shape, generator=torch.Generator().manual_seed(k)).to(dev)
        way /= way.norm()
        f = [slk.linear_cross_entropy(h + s * step * way if k == 0 else h,
                                      w + s * step * way if k == 1 else w, t, reduction="none")
             .double().mean() for s in (1, -1)]
        assert abs(float(f[0] - f[1]) / (2 * step) - float((g * way).sum())) \
            < step * step * 512 / n + 2.0 ** -14


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_another_ignore_index_and_leading_sizes(dev, dtype, n, d, v):
    h, w, t = make(n, d, v, dtype, dev, 5)
    t[::5] = 0
    h.requires_grad_()
    a = slk.linear_cross_entropy(h.reshape(2, n // 2, d), w, t.reshape(2, n // 2),
                                 ignore_index=0, reduction="none")
    losses, err, dh, eh, _, _ = reference(h, w, t, torch.ones(n, device=dev), ignore=0)
    assert a.shape == (2, n // 2)
    within(a.reshape(-1), losses, err, "loss")
    gh, = torch.autograd.grad(a, h, torch.ones_like(a))
    within(gh, dh, eh, "dh")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_row_of_dw_over_several_pieces(dev, dtype):
    """More logits than one piece of the backward holds, every row of dw compared: wherever
    the pieces end (three in float32, two in bfloat16)."""
    from sparsecore_amd import _lib

    n, d, v = 8192, 48, 40000
    a = _lib.LinearCE(n=n, d=d, v=v, dtype=_lib.DTYPES[dtype], reduction=1, keep=1, dhidden=16,
                      dweight=16)
    assert _lib.linear_ce_scratch_bytes(a, True) < n * v * 4  # not all of dl
    h, w, t = make(n, d, v, dtype, dev, 6, 0.1)
    h.requires_grad_(), w.requires_grad_()
    loss = slk.linear_cross_entropy(h, w, t, reduction="sum")
    gh, gw = torch.autograd.grad(loss, [h, w])
    hd, wd = h.detach().double(), w.detach().double()
    live = (t != -100)[:, None]
    lse = torch.cat([torch.logsumexp(x @ wd.t(), 1) for x in hd.split(512)])[:, None]
    for lo in range(0, v, 5000):
        rows = slice(lo, lo + 5000)
        p = torch.exp(hd @ wd[rows].t() - lse)
        hit = (t[:, None] == torch.arange(v, device=dev)[rows]) & live
        dl = torch.where(live, p - hit.double(), 0.0)
        want = dl.t() @ hd
        terms = dl.abs().t() @ hd.abs()
        tol = (2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -17) * terms
        within(gw[rows], want, tol + 2.0 ** -8 * want.abs() * (dtype is torch.bfloat16),
               f"dw from {lo}")
