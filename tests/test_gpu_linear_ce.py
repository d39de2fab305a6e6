"""linear_cross_entropy against its definition in float64, and its gradient against
differences.

Bounds, with S = Σ_k |h_k w_k| of a logit. A float32 operand is kept to 2^-22 of itself,
the product of the two low parts is dropped (2^-22) and the sum is float32: a logit is off
by e_z = 2^-20 S at most (bfloat16 operands: exact products, the same sum). A loss is then
off by 2 max e_z and its own rounding. A softmax entry p is off by 2 p max e_z and a few
units of p, dl = p - onehot is kept to 2^-38 of 1 (float32) or 2^-8 of itself
(bfloat16), and the gradients are sums of |dl error| · |operand| plus 2^-20 of their own
terms' absolute sum; bfloat16 results round once more, by 2^-8 at most.
"""

from __future__ import annotations

import math

import pytest
import torch

import sparsecore_amd as slk

pytestmark = pytest.mark.gpu

E = 2.0 ** -20


def make(n, d, v, dtype, dev, seed=0, ignored=0.0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    h = (torch.randn(n, d, generator=g) * scale).to(dtype)
    w = (torch.randn(v, d, generator=g) * 2 / math.sqrt(d)).to(dtype)
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.rand(n, generator=g) < ignored] = -100
    return h.to(dev), w.to(dev), t.to(dev)


def reference(h, w, t, up, ignore=-100):
    """(losses, dh, dw, and their bounds) for upstream gradients `up` of each token."""
    dtype = h.dtype
    h, w, t, up = h.detach().double(), w.detach().double(), t, up.double()
    live = t != ignore
    h = torch.where(live[:, None], h, 0.0)
    z = h @ w.t()
    ez = 2 * E * (h.abs() @ w.abs().t()).amax(1, keepdim=True) if w.numel() else z
    lse = torch.logsumexp(z, 1, keepdim=True)
    idx = torch.where(live, t, 0)[:, None]
    losses = torch.where(live, (lse - z.gather(1, idx)).squeeze(1), 0.0)
    loss_err = torch.where(live, ez.squeeze(1) + 2e-6 * (1 + lse.squeeze(1).abs()
                                                        + z.gather(1, idx).squeeze(1).abs()), 0.0)
    p = torch.exp(z - lse)
    dl = p.scatter_add(1, idx, -torch.ones_like(lse))
    err = p * (ez + 2e-6) + 2.0 ** -38
    if dtype is torch.bfloat16:
        err = err + 2.0 ** -8 * dl.abs()
    g = torch.where(live, up, 0.0)[:, None]
    top = g.abs().max() if g.numel() else 0.0
    dl, err = dl * g, torch.where(live[:, None], err * g.abs() + 2.0 ** -38 * top, 0.0)
    dh, dw = dl @ w, dl.t() @ h
    dh_err = err @ w.abs() + E * (dl.abs() @ w.abs())
    dw_err = err.t() @ h.abs() + E * (dl.abs().t() @ h.abs())
    if dtype is torch.bfloat16:
        dh_err, dw_err = dh_err + 2.0 ** -8 * dh.abs(), dw_err + 2.0 ** -8 * dw.abs()
    return losses, loss_err, dh, dh_err, dw, dw_err


def within(got, want, err, what):
    got = got.detach().double()
    assert got.shape == want.shape, what
    far = (got - want).abs() - err
    assert bool((far <= 0).all()), f"{what}: {float(far.max()):.3g} beyond"


def check(dev, n, d, v, dtype, ignored=0.0, reduction="mean", seed=0, scale=1.0):
    h, w, t = make(n, d, v, dtype, dev, seed, ignored, scale)
    h.requires_grad_(), w.requires_grad_()
    loss = slk.linear_cross_entropy(h, w, t, reduction=reduction)
    live = int((t != -100).sum())
    if reduction == "none":
        up = torch.randn(n, generator=torch.Generator().manual_seed(9)).to(dev)
        losses, lerr, dh, eh, dw, ew = reference(h, w, t, up)
        within(loss, losses, lerr, "loss")
    else:
        up = torch.tensor(0.37, device=dev)
        share = 0.37 / live if reduction == "mean" and live else 0.37
        each = torch.full((n,), share, dtype=torch.float64, device=dev)
        losses, lerr, dh, eh, dw, ew = reference(h, w, t, each)
        if reduction == "mean" and not live:
            assert bool(torch.isnan(loss))
        else:
            by = live if reduction == "mean" else 1
            within(loss, losses.sum() / by, lerr.sum() / by + 1e-6 * losses.sum() / by, "loss")
        eh, ew = eh + 2e-7 * dh.abs(), ew + 2e-7 * dw.abs()  # the factor's rounding
    gh, gw = torch.autograd.grad(loss, [h, w], up)
    within(gh, dh, eh, "dh")
    within(gw, dw, ew, "dw")
    assert gh.dtype == dtype and gw.dtype == dtype


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", [(1, 1, 1), (1, 64, 65), (2, 3, 2), (31, 32, 33), (128, 64, 256),
                                   (129, 65, 257), (300, 200, 1000), (1000, 384, 65),
                                   (65, 1000, 4099), (513, 96, 513)])
def test_sizes(dev, dtype, n, d, v):
    check(dev, n, d, v, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("ignored", [0.0, 0.3, 0.97, 1.0])
def test_reductions_and_ignored_tokens(dev, dtype, reduction, ignored):
    check(dev, 200, 80, 300, dtype, ignored, reduction)
    check(dev, 1, 80, 300, dtype, ignored, reduction)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_tokens_and_a_large_vocabulary(dev, dtype):
    check(dev, 9000, 64, 300, dtype, 0.2)
    check(dev, 70, 128, 33000, dtype, 0.2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces_of_the_vocabulary(dev, dtype):
    """More logits than a piece of the backward holds: 2^30 bytes of logit gradients are
    8192 x 16384 in float32 and twice as many in bfloat16."""
    n, d, v = 8192, 48, 40000
    h, w, t = make(n, d, v, dtype, dev, 1, 0.1)
    h.requires_grad_(), w.requires_grad_()
    loss = slk.linear_cross_entropy(h, w, t, reduction="sum")
    gh, gw = torch.autograd.grad(loss, [h, w])
    for lo in (0, 16384 - 100, 32768 - 100, v - 100):  # rows of dw around the pieces' ends
        rows = slice(lo, lo + 200)
        z = h.detach().double() @ w.detach().double().t()
        p = torch.exp(z[:, rows] - torch.logsumexp(z, 1, keepdim=True))
        del z
        live = (t != -100)[:, None]
        hit = (t[:, None] == torch.arange(v, device=dev)[rows]) & live
        dl = torch.where(live, p - hit.double(), 0.0)
        want = dl.t() @ h.detach().double()
        terms = dl.abs().t() @ h.detach().double().abs()
        tol = (2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -17) * terms \
            + 2.0 ** -38 * h.detach().double().abs().sum(0)
        within(gw[rows], want, tol + 2.0 ** -8 * want.abs() * (dtype is torch.bfloat16), "dw")
    some = torch.arange(0, n, 331, device=dev)
    _, _, dh, eh, _, _ = reference(h[some], w, t[some], torch.ones(len(some), device=dev))
    within(gh[some], dh, eh, "dh")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 15, 16, 17])
@pytest.mark.parametrize("d,v", [(1, 3), (40, 17), (100, 1), (768, 5000), (130, 777)])
def test_scores_of_a_few_tokens(dev, dtype, n, d, v):
    h, w, t = make(n, d, v, dtype, dev, 2)
    if n > 2:
        t[1] = -100
    got = slk.linear_cross_entropy(h, w, t, reduction="none")
    losses, err, *_ = reference(h, w, t, torch.zeros(n, device=dev))
    within(got, losses, err, "loss")
    mean = slk.linear_cross_entropy(h, w, t)
    live = int((t != -100).sum())
    within(mean, losses.sum() / live, err.sum() / live + 1e-6 * losses.sum() / live, "mean")


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 30.0, 1e4])
def test_ranges_of_float32(dev, scale):
    """Hidden states far from 1 keep their relative precision (the power-of-two scaling);
    at 30 and 1e4 the softmax is one-hot."""
    check(dev, 100, 64, 200, torch.float32, scale=scale)


def test_small_rows_beside_large_ones(dev):
    """Rows a thousandth of the largest: every logit stays within its own bound."""
    h, w, t = make(64, 96, 300, torch.float32, dev, 3)
    h = h * torch.logspace(-3, 1, 64, device=dev)[:, None]
    losses, err, *_ = reference(h, w, t, torch.zeros(64, device=dev))
    within(slk.linear_cross_entropy(h, w, t, reduction="none"), losses, err, "loss")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_ignored_tokens_reach_nothing(dev, dtype, bad):
    h, w, t = make(50, 64, 100, dtype, dev, 4)
    t[::3] = -100
    h[::3] = bad
    h.requires_grad_(), w.requires_grad_()
    loss = slk.linear_cross_entropy(h, w, t)
    gh, gw = torch.autograd.grad(loss, [h, w])
    up = torch.full((50,), 1.0 / int((t != -100).sum()), dtype=torch.float64, device=dev)
    losses, lerr, dh, eh, dw, ew = reference(h, w, t, up)
    count = int((t != -100).sum())
    within(loss, losses.sum() / count, lerr.sum() / count + 1e-6, "loss")
    within(gh, dh, eh + 2e-7 * dh.abs(), "dh")
    within(gw, dw, ew + 2e-7 * dw.abs(), "dw")
    assert bool((gh[::3] == 0).all())


def test_a_live_nan_stays_in_its_loss_and_dh(dev):
    h, w, t = make(40, 64, 100, torch.float32, dev, 5)
    clean = slk.linear_cross_entropy(h, w, t, reduction="none")
    h[7, 3] = float("nan")
    h.requires_grad_()
    got = slk.linear_cross_entropy(h, w, t, reduction="none")
    keep = torch.arange(40, device=dev) != 7
    torch.testing.assert_close(got[keep], clean[keep], rtol=1e-6, atol=1e-6)
    assert bool(torch.isnan(got[7]))
    gh, = torch.autograd.grad(got, h, torch.ones_like(got))
    assert bool(torch.isfinite(gh[keep]).all()) and bool(torch.isnan(gh[7]).all())


def test_targets_outside_the_vocabulary(dev):
    for n in (8, 40):
        h, w, t = make(n, 64, 100, torch.float32, dev, 6)
        clean = slk.linear_cross_entropy(h, w, t, reduction="none")
        t[2], t[5] = 100, -7
        got = slk.linear_cross_entropy(h, w, t, reduction="none")
        assert bool(torch.isnan(got[[2, 5]]).all())
        keep = [i for i in range(n) if i not in (2, 5)]
        assert torch.equal(got[keep], clean[keep])
        h.requires_grad_(), w.requires_grad_()
        loss = slk.linear_cross_entropy(h, w, t)
        assert bool(torch.isnan(loss))
        gh, gw = torch.autograd.grad(loss, [h, w])
        assert bool(torch.isfinite(gh).all()) and bool(torch.isfinite(gw).all())


def test_another_ignore_index_and_leading_sizes(dev):
    h, w, t = make(24, 64, 100, torch.float32, dev, 7)
    t[3] = 0
    a = slk.linear_cross_entropy(h.reshape(2, 12, 64), w, t.reshape(2, 12), ignore_index=0,
                                 reduction="none")
    losses, err, *_ = reference(h, w, t, torch.zeros(24, device=dev), ignore=0)
    assert a.shape == (2, 12)
    within(a.reshape(-1), losses, err, "loss")


def test_gradient_against_differences(dev):
    """Central differences along random directions, step 2^-6: truncation h² times a
    third derivative of order 1 (2e-4), rounding about 2^-20 / h (6e-5)."""
    h, w, t = make(20, 32, 50, torch.float32, dev, 8)
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    grads = torch.autograd.grad(slk.linear_cross_entropy(hg, wg, t), [hg, wg])
    step = 2.0 ** -6
    for k, g in enumerate(grads):
        way = torch.randn(g.shape, generator=torch.Generator().manual_seed(k)).to(dev)
        way /= way.norm()
        f = [slk.linear_cross_entropy(h + s * step * way * (k == 0) if k == 0 else h,
                                      w + s * step * way if k == 1 else w, t, reduction="none")
             .double().mean() for s in (1, -1)]
        assert abs(float(f[0] - f[1]) / (2 * step) - float((g * way).sum())) < 3e-4


def test_results_repeat_and_other_streams(dev):
    h, w, t = make(700, 200, 900, torch.float32, dev, 9, 0.2)
    h.requires_grad_(), w.requires_grad_()

    def once():
        loss = slk.linear_cross_entropy(h, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, [h, w]))

    a = once()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = once()
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_one_gradient_alone_and_none(dev):
    h, w, t = make(100, 64, 300, torch.float32, dev, 10)
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(slk.linear_cross_entropy(hg, wg, t), [hg, wg])
    one, = torch.autograd.grad(slk.linear_cross_entropy(hg, w, t), hg)
    other, = torch.autograd.grad(slk.linear_cross_entropy(h, wg, t), wg)
    assert torch.equal(one, both[0]) and torch.equal(other, both[1])
    assert not slk.linear_cross_entropy(h, w, t).requires_grad


def test_no_tokens(dev):
    h = torch.zeros(0, 64, device=dev, requires_grad=True)
    w = torch.ones(10, 64, device=dev, requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device=dev)
    loss = slk.linear_cross_entropy(h, w, t, reduction="sum")
    loss.backward()
    assert float(loss) == 0 and bool((w.grad == 0).all()) and h.grad.shape == (0, 64)
    assert bool(torch.isnan(slk.linear_cross_entropy(h, w, t)))


def test_refusals(dev):
    h, w, t = make(4, 8, 10, torch.float32, dev)
    f = slk.linear_cross_entropy
    with pytest.raises(TypeError):
        f(h, w, [1, 2, 3, 4])
    with pytest.raises(RuntimeError, match="HIP"):
        f(h.cpu(), w, t)
    with pytest.raises(RuntimeError, match="HIP"):
        f(h, w, t.cpu())
    with pytest.raises(ValueError, match="reduction"):
        f(h, w, t, reduction="max")
    with pytest.raises(ValueError, match="int64"):
        f(h, w, t.int())
    with pytest.raises(ValueError, match="float32 or both"):
        f(h, w.bfloat16(), t)
    with pytest.raises(ValueError, match="float32 or both"):
        f(h.half(), w.half(), t)
    for bad in ((h[:, :7], w, t), (h, w, t[:3]), (h, w[0], t), (h[0], w, t)):
        with pytest.raises(ValueError):
            f(*bad)


def test_scores_without_gradients_keep_nothing(dev, monkeypatch):
    """Under no_grad the head's own requires_grad must not cost the packed operands."""
    from sparsecore_amd import _lib

    h, w, t = make(8, 64, 300, torch.float32, dev, 11)
    w.requires_grad_()
    seen = []
    real = _lib.linear_ce_forward
    monkeypatch.setattr(_lib, "linear_ce_forward", lambda a, s: (seen.append(a.keep), real(a, s)))
    with torch.no_grad():
        slk.linear_cross_entropy(h, w, t)
    slk.linear_cross_entropy(h, w, t)
    assert seen == [0, 1]


def test_double_backward_is_refused(dev):
    h, w, t = make(8, 64, 300, torch.float32, dev, 12)
    h.requires_grad_()
    up = torch.ones((), device=dev, requires_grad=True)
    g, = torch.autograd.grad(slk.linear_cross_entropy(h, w, t), h, up, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", [(1, 1, 1), (5, 33, 70), (300, 130, 517), (16, 50, 300)])
@pytest.mark.parametrize("keep", [0, 1])
def test_writes_stay_in_range(dev, dtype, n, d, v, keep):
    """Through the C-ABI with guard bytes around every array that it may write."""
    from sparsecore_amd import _lib

    h, w, t = make(n, d, v, dtype, dev, 13, 0.3)
    size = h.element_size()
    args = _lib.LinearCE(n=n, d=d, v=v, ignore_index=-100, hidden=h.data_ptr(),
                         weight=w.data_ptr(), target=t.data_ptr(), dtype=_lib.DTYPES[dtype],
                         reduction=0, keep=keep)
    up = torch.ones(n, device=dev)

    def guarded(nbytes):
        buf = torch.full((nbytes + 1024,), 0xA5, dtype=torch.uint8, device=dev)
        return buf, buf.data_ptr() + 512

    def intact(buf):
        return bool((buf[:512] == 0xA5).all()) and bool((buf[-512:] == 0xA5).all())

    def up256(x):  # addresses of the workspaces keep torch's alignment
        return (x + 255) // 256 * 256

    loss, args.loss = guarded(4 * n)
    args.saved_bytes = _lib.linear_ce_saved_bytes(args)
    args.scratch_bytes = _lib.linear_ce_scratch_bytes(args, False)
    saved, args.saved = guarded(up256(args.saved_bytes))
    scratch, args.scratch = guarded(up256(args.scratch_bytes))
    _lib.linear_ce_forward(args, _lib.stream_of(h))
    torch.cuda.synchronize()
    assert intact(loss) and intact(saved) and intact(scratch)
    if not keep:
        return
    dh, args.dhidden = guarded(size * n * d)
    dw, args.dweight = guarded(size * v * d)
    args.upstream = up.data_ptr()
    args.scratch_bytes = _lib.linear_ce_scratch_bytes(args, True)
    scratch, args.scratch = guarded(up256(args.scratch_bytes))
    _lib.linear_ce_backward(args, _lib.stream_of(h))
    torch.cuda.synchronize()
    assert all(intact(b) for b in (dh, dw, saved, scratch))


def test_captured_loss_and_gradients_replay(dev):
    h, w, t = make(300, 64, 500, torch.float32, dev, 14, 0.2)
    h.requires_grad_(), w.requires_grad_()

    def once():
        loss = slk.linear_cross_entropy(h, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, [h, w]))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        got = once()
    from sparsecore_amd import _lib

    assert "memset" not in _lib.graph_node_types(graph)
    graph.instantiate()
    for k in range(4):
        with torch.no_grad():
            h.copy_(torch.randn(300, 64, generator=torch.Generator().manual_seed(k)))
            t.copy_(torch.where(torch.rand(300, generator=torch.Generator().manual_seed(k)) < 0.1 * k,
                                -100, torch.randint(0, 500, (300,))))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, once()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [2, 16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("d,v", [(4, 31), (63, 32), (64, 33), (257, 500), (520, 3001)])
def test_gradients_of_few_tokens(dev, dtype, n, d, v):
    check(dev, n, d, v, dtype, 0.2, "mean" if n % 2 else "none")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [32, 33, 64, 100, 128, 129])
@pytest.mark.parametrize("d,v", [(72, 100), (100, 3001), (1030, 70)])
def test_scores_of_some_tokens(dev, dtype, n, d, v):
    h, w, t = make(n, d, v, dtype, dev, 20, 0.2)
    losses, err, *_ = reference(h, w, t, torch.zeros(n, device=dev))
    within(slk.linear_cross_entropy(h, w, t, reduction="none"), losses, err, "loss")


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 30.0, 1e4])
def test_ranges_of_float32_few_tokens(dev, scale):
    check(dev, 30, 64, 200, torch.float32, scale=scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_few_ignored_tokens_reach_nothing(dev, dtype, bad):
    h, w, t = make(25, 64, 100, dtype, dev, 21)
    clean = torch.where(torch.arange(25, device=dev)[:, None] % 3 == 0, 0, h)
    t[::3] = -100
    grads = []
    for x in (torch.where(torch.arange(25, device=dev)[:, None] % 3 == 0, bad, h), clean):
        x, y = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = slk.linear_cross_entropy(x, y, t)
        grads.append((loss.detach(), *torch.autograd.grad(loss, [x, y])))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    assert bool((grads[0][1][::3] == 0).all()) and bool(torch.isfinite(grads[0][2]).all())


def test_few_tokens_one_gradient_alone_alignment_and_targets(dev):
    h, w, t = make(40, 64, 300, torch.float32, dev, 22)
    t[3], t[9] = 300, -5  # no rows of the vocabulary

    def grads(h, w):
        want = [x for x in (h, w) if x.requires_grad]
        return torch.autograd.grad(slk.linear_cross_entropy(h, w, t), want)

    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    both = grads(hg, wg)
    assert torch.equal(grads(hg, w)[0], both[0]) and torch.equal(grads(h, wg)[0], both[1])
    assert bool(torch.isfinite(both[0]).all()) and bool(torch.isfinite(both[1]).all())
    odd = torch.empty(h.numel() + 1, device=dev)[1:].view_as(h).copy_(h).requires_grad_()
    torch.testing.assert_close(grads(odd, w)[0], both[0], rtol=1e-5, atol=1e-7)


def test_few_tokens_refuse_a_weight_that_changed(dev):
    """Their backward reads weight itself, so autograd must hold its version."""
    h, w, t = make(8, 64, 100, torch.float32, dev, 23)
    h.requires_grad_()
    loss = slk.linear_cross_entropy(h, w, t)
    w.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_captured_few_tokens_replay(dev):
    h, w, t = make(20, 64, 500, torch.float32, dev, 24, 0.2)
    h.requires_grad_(), w.requires_grad_()

    def once():
        loss = slk.linear_cross_entropy(h, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, [h, w]))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for k in range(4):
        with torch.no_grad():
            h.copy_(torch.randn(20, 64, generator=torch.Generator().manual_seed(k)))
            t.copy_(torch.randint(0, 500, (20,), generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, once()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 16, 65, 80, 81, 128, 129])
@pytest.mark.parametrize("n,d", [(65, 4), (129, 63), (300, 260), (1000, 520), (5000, 64)])
def test_small_vocabularies(dev, dtype, v, n, d):
    check(dev, n, d, v, dtype, 0.2, ("mean", "none", "sum")[n % 3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_small_vocabularys_ignored_tokens_reach_nothing(dev, dtype, bad):
    h, w, t = make(500, 70, 65, dtype, dev, 25)
    t[::3] = -100
    at = (torch.arange(500, device=dev) % 3 == 0)[:, None]
    runs = []
    for x in (torch.where(at, bad, h), torch.where(at, 0, h)):
        x, y = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = slk.linear_cross_entropy(x, y, t)
        runs.append((loss.detach(), *torch.autograd.grad(loss, [x, y])))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert bool((runs[0][1][::3] == 0).all()) and bool(torch.isfinite(runs[0][2]).all())


def test_a_small_vocabularys_gradients_alone_targets_and_captures(dev):
    h, w, t = make(700, 64, 65, torch.float32, dev, 26, 0.2)
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()

    def once(h, w):
        loss = slk.linear_cross_entropy(h, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, [x for x in (h, w) if x.requires_grad]))

    both = once(hg, wg)
    assert torch.equal(once(hg, w)[1], both[1]) and torch.equal(once(h, wg)[1], both[2])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once(hg, wg)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once(hg, wg)
    for k in range(4):
        with torch.no_grad():
            hg.copy_(torch.randn(700, 64, generator=torch.Generator().manual_seed(k)))
            t.copy_(torch.randint(0, 65, (700,), generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, once(hg, wg)))
    t[3], t[9] = 65, -5  # no rows of the vocabulary
    loss, gh, gw = once(hg, wg)
    assert bool(torch.isnan(loss)) and bool(torch.isfinite(gh).all() & torch.isfinite(gw).all())


@pytest.mark.parametrize("keep", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,v", [(130, 33, 70), (65, 260, 128), (40, 50, 300), (64, 257, 31)])
def test_unpacked_writes_stay_in_range(dev, dtype, n, d, v, keep):
    test_writes_stay_in_range(dev, dtype, n, d, v, keep)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [12, 30, 60, 128])
@pytest.mark.parametrize("ignored", [0.6, 0.95, 1.0])
def test_few_tokens_mostly_ignored(dev, dtype, n, ignored):
    h, w, t = make(n, 200, 700, dtype, dev, 27, ignored)
    losses, err, *_ = reference(h, w, t, torch.zeros(n, device=dev))
    within(slk.linear_cross_entropy(h, w, t, reduction="none"), losses, err, "loss")
    check(dev, n, 200, 700, dtype, ignored, "none", 27)
