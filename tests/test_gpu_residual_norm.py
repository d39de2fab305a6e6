"""residual_norm against its definition in float64, with autograd's float64 gradients,
and its gradient against differences.

Bounds. Every result is a sum of terms that may cancel (a LayerNorm of one feature has the
gradient 0), so errors are measured against the terms: `magnitudes` adds the absolute
values of the formula's terms in float64. A float32 sum of them is off by at most
(terms + 12) u of that sum, u = 2^-24, and by far less with roundings that do not all
point one way: 1e-5 of the magnitude's root mean square holds for every size here.
bfloat16 results are rounded once, 2^-9 relative (2^-8 taken), and the backward reads back
the rounded r, 2^-9 of xhat: 3 · 2^-8 of the magnitude covers both norms.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import sparsecore_amd as slk
from sparsecore_amd import _lib

pytestmark = pytest.mark.gpu


def make(shape, d, kind, post, gate, dtype, dev, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)

    def rand(*s, scale=1.0, mean=0.0):
        return (mean + scale * torch.randn(*s, generator=g)).to(dtype).to(dev)

    n = 1
    for k in shape:
        n *= k
    t = {"x": rand(*shape, d, scale=2.0, mean=0.3), "branch": rand(*shape, d),
         "weight": rand(d, scale=0.2, mean=1.0)}
    if kind == "layer" and bias:
        t["bias"] = rand(d, scale=0.2)
    if post:
        t["post_weight"] = rand(d, scale=0.2, mean=1.0)
        if kind == "layer" and bias:
            t["post_bias"] = rand(d, scale=0.2)
    if gate == "feature":
        t["gate"] = rand(d, scale=0.5)
    elif gate == "element":
        t["gate"] = rand(*shape, d, scale=0.5)
    elif gate == "sequence":
        t["gate"] = rand(shape[0], *([1] * (len(shape) - 1)), d, scale=0.5)
    return t, rand(*shape, d), rand(*shape, d)


def reference(t, kind, scale, eps):
    d = t["x"].shape[-1]

    def norm(v, w, b):
        if kind == "layer":
            return F.layer_norm(v, (d,), t[w], t.get(b), eps)
        return F.rms_norm(v, (d,), t[w], eps)

    if "branch" not in t:
        return t["x"], norm(t["x"], "weight", "bias")
    o = norm(t["branch"], "post_weight", "post_bias") if "post_weight" in t else t["branch"]
    r = t["x"] + scale * (o * t["gate"] if "gate" in t else o)
    return r, norm(r, "weight", "bias")


def magnitudes(t, dr, dy, kind, scale, eps):
    """For r, y and every gradient: the sum of the absolute values of its terms."""
    t = {k: v.detach().double().cpu() for k, v in t.items()}
    dr, dy = dr.double().cpu(), dy.double().cpu()
    d = t["x"].shape[-1]

    def stats(v):
        mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
        rstd = 1 / ((v - mean).square().mean(-1, keepdim=True) + eps).sqrt()
        return (v.abs() + abs(mean)) * rstd, rstd  # (v - mean) · rstd, before cancelling

    def back(g, xhat, rstd):
        return rstd * (g + g.mean(-1, keepdim=True) + xhat * (g * xhat).mean(-1, keepdim=True))

    one = torch.ones(())
    gate = t.get("gate", one).abs()
    o = t["branch"].abs()
    if "post_weight" in t:
        uhat, urstd = stats(t["branch"])
        o = uhat * t["post_weight"].abs() + t.get("post_bias", one * 0).abs()
    m = {"r": t["x"].abs() + abs(scale) * gate * o}
    xhat, rstd = stats(reference(t, kind, scale, eps)[0])
    m["y"] = xhat * t["weight"].abs() + t.get("bias", one * 0).abs()
    g = dr.abs() + back(dy.abs() * t["weight"].abs(), xhat, rstd)
    m["dx"] = g
    flat = tuple(range(dy.dim() - 1))
    m["dweight"], m["dbias"] = (dy.abs() * xhat).sum(flat), dy.abs().sum(flat)
    b = abs(scale) * g * gate
    if "gate" in t:
        m["dgate"] = abs(scale) * g * o
        shared = [i for i, k in enumerate(t["gate"].shape) if k == 1 and g.shape[i] != 1]
        if t["gate"].dim() == 1:
            m["dgate"] = m["dgate"].sum(flat)
        elif shared and t["gate"].shape != g.shape:
            m["dgate"] = m["dgate"].sum(shared, keepdim=True)
    m["dbranch"] = b
    if "post_weight" in t:
        m["dpost_weight"], m["dpost_bias"] = (b * uhat).sum(flat), b.sum(flat)
        m["dbranch"] = back(b * t["post_weight"].abs(), uhat, urstd)
    return m


def close(got, want, dtype, what, mag=None):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, what
    mag = want.abs() if mag is None else mag
    assert mag.shape == want.shape, what
    rms = mag.square().mean().sqrt()
    tol = 1e-5 * (rms + mag) if dtype is torch.float32 else 2.0 ** -8 * mag + 3 * 2.0 ** -8 * rms
    worst = ((got - want).abs() - tol).max() if got.numel() else torch.tensor(-1.0)
    assert float(worst) <= 0, f"{what}: {float(worst):.3g} beyond, rms {float(rms):.3g}"


def cols(t):
    d = t.shape[-1]
    return t.reshape(-1, d).t().contiguous().t().reshape(t.shape)


def check(dev, shape, d, kind, post, gate, dtype, cols_in=False, cols_out=False, bias=True,
          scale=0.7, offset=0):
    eps = 1e-5
    t, dr, dy = make(shape, d, kind, post, gate, dtype, dev, bias=bias)
    if offset:
        t = {k: torch.cat([v.new_zeros(offset), v.reshape(-1)])[offset:].view(v.shape)
             for k, v in t.items()}
    if cols_in:
        t["branch"], dy = cols(t["branch"]), cols(dy)
    ref = {k: v.detach().double().cpu().requires_grad_() for k, v in t.items()}
    for v in t.values():
        v.requires_grad_()
    args = {k: v for k, v in t.items() if k not in ("x", "weight", "bias")}
    r, y = slk.residual_norm(t["x"], t["weight"], t.get("bias"), scale=scale, kind=kind, eps=eps,
                             feature_major=cols_out, **args)
    rr, ry = reference(ref, kind, scale, eps)
    mag = magnitudes(t, dr, dy, kind, scale, eps)
    close(r, rr, dtype, "r", mag["r"])
    close(y, ry, dtype, "y", mag["y"])
    if cols_out:
        assert y.reshape(-1, d).t().is_contiguous()
    got = torch.autograd.grad([r, y], list(t.values()), [dr, dy])
    want = torch.autograd.grad([rr, ry], list(ref.values()), [dr.double().cpu(),
                                                              dy.double().cpu()])
    for k, a, b in zip(t, got, want):
        close(a, b, dtype, "d" + k, mag["d" + k])
    if cols_in:
        assert got[list(t).index("branch")].reshape(-1, d).t().is_contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("d", [1, 2, 63, 64, 384, 513, 768, 1001, 1024, 1500, 2048, 4096, 5000,
                               8192, 12001, 16384])
def test_widths(dev, dtype, kind, d):
    check(dev, (13,), d, kind, True, "feature", dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["none", "feature", "sequence", "element"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("shape", [(1,), (2, 1), (7, 5), (3, 700), (2, 3, 11)])
@pytest.mark.parametrize("d", [96, 1300])
def test_gates_and_post_norms(dev, dtype, gate, post, shape, d):
    check(dev, shape, d, "layer", post, gate, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["none", "feature", "sequence", "element"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("shape", [(1,), (15,), (16,), (2, 33), (4, 256)])
@pytest.mark.parametrize("d", [1, 65, 384, 1000, 1024, 1100])
def test_feature_major(dev, dtype, gate, post, shape, d):
    check(dev, shape, d, "layer", post, gate, dtype, cols_in=True, cols_out=True)


@pytest.mark.parametrize("cols_in,cols_out", [(True, False), (False, True)])
def test_one_side_feature_major(dev, cols_in, cols_out):
    check(dev, (5, 40), 320, "rms", True, "sequence", torch.float32, cols_in, cols_out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_odd_alignment_and_no_bias(dev, dtype):
    check(dev, (9, 4), 128, "layer", True, "element", dtype, offset=1)
    check(dev, (9, 4), 128, "layer", True, "none", dtype, bias=False)


def test_many_tokens_sum_in_a_fixed_order(dev):
    check(dev, (4, 5000), 96, "layer", True, "sequence", torch.float32)
    t, dr, dy = make((6, 3000), 200, "layer", True, "sequence", torch.float32, dev)
    for v in t.values():
        v.requires_grad_()
    args = {k: v for k, v in t.items() if k not in ("x", "weight", "bias")}
    runs = []
    for _ in range(2):
        r, y = slk.residual_norm(t["x"], t["weight"], t["bias"], **args)
        runs.append(torch.autograd.grad([r, y], list(t.values()), [dr, dy]))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_no_branch(dev, kind):
    t, _, dy = make((3, 50), 96, kind, False, "none", torch.float32, dev)
    del t["branch"]
    ref = {k: v.double().cpu().requires_grad_() for k, v in t.items()}
    for v in t.values():
        v.requires_grad_()
    r, y = slk.residual_norm(t["x"], t["weight"], t.get("bias"), kind=kind)
    assert r is t["x"]
    got = torch.autograd.grad(y, list(t.values()), dy)
    want = torch.autograd.grad(reference(ref, kind, 1.0, 1e-5)[1], list(ref.values()),
                               dy.double().cpu())
    for k, a, b in zip(t, got, want):
        close(a, b, torch.float32, "d" + k)


def test_gradient_of_one_output_alone(dev):
    t, dr, dy = make((4, 9), 96, "layer", True, "sequence", torch.float32, dev)
    for v in t.values():
        v.requires_grad_()
    args = {k: v for k, v in t.items() if k not in ("x", "weight", "bias")}
    for which in (0, 1):
        ref = {k: v.detach().double().cpu().requires_grad_() for k, v in t.items()}
        out = slk.residual_norm(t["x"], t["weight"], t["bias"], **args)[which]
        want = reference(ref, "layer", 1.0, 1e-5)[which]
        up = (dr, dy)[which]
        got = torch.autograd.grad(out, list(t.values()), up, allow_unused=True)
        want = torch.autograd.grad(want, list(ref.values()), up.double().cpu(),
                                   allow_unused=True)
        for k, a, b in zip(t, got, want):
            close(a, torch.zeros_like(ref[k]) if b is None else b, torch.float32, "d" + k)


def test_gradients_not_asked_for_are_not_needed(dev):
    t, dr, dy = make((4, 9), 96, "layer", True, "sequence", torch.float32, dev)
    args = {k: v for k, v in t.items() if k not in ("x", "weight", "bias")}
    ref = {k: v.double().cpu() for k, v in t.items()}
    for name in t:
        t[name].requires_grad_()
        ref[name].requires_grad_()
        r, y = slk.residual_norm(t["x"], t["weight"], t["bias"], **args)
        rr, ry = reference(ref, "layer", 1.0, 1e-5)
        ours, theirs = [r, y], [rr, ry]
        if not r.requires_grad or not rr.requires_grad:
            ours, theirs = [y], [ry]
        ups = [dr, dy][-len(ours):]
        got, = torch.autograd.grad(ours, t[name], ups, allow_unused=True)
        want, = torch.autograd.grad(theirs, ref[name], [u.double().cpu() for u in ups])
        close(got, want, torch.float32, "d" + name)
        t[name].requires_grad_(False)
        ref[name].requires_grad_(False)


def test_gradient_against_differences(dev):
    """Central differences of Σ(r·dr + y·dy) along random directions, h = 2^-7: the
    truncation is h² times a third derivative of order 1, the rounding about 2^-24 ·
    |sum's terms| / h, both below 2e-3 of the directional derivative's scale here."""
    t, dr, dy = make((6,), 64, "layer", True, "element", torch.float32, dev)
    args = ("branch", "gate", "post_weight", "post_bias")

    def f(p):
        r, y = slk.residual_norm(p["x"], p["weight"], p["bias"], scale=0.7,
                                 **{k: p[k] for k in args})
        return (r.double() * dr.double()).sum() + (y.double() * dy.double()).sum()

    p = {k: v.clone().requires_grad_() for k, v in t.items()}
    grads = torch.autograd.grad(f(p), list(p.values()))
    h = 2.0 ** -7
    for (k, v), g in zip(t.items(), grads):
        way = torch.randn(v.shape, generator=torch.Generator().manual_seed(3)).to(dev)
        hi, lo = ({**t, k: v + s * h * way} for s in (1, -1))
        slope = float(f(hi) - f(lo)) / (2 * h)
        want = float((g.double() * way.double()).sum())
        scale = float((g.double() * way.double()).square().sum().sqrt())
        assert abs(slope - want) <= 2e-3 * max(1.0, abs(want), scale), k


def test_rows_keep_to_themselves(dev):
    """NaN and infinities of one token reach no other token's results."""
    t, _, _ = make((40,), 200, "layer", True, "element", torch.float32, dev)
    args = {k: v for k, v in t.items() if k not in ("x", "weight", "bias")}
    clean = slk.residual_norm(t["x"], t["weight"], t["bias"], **args)
    for bad in (float("nan"), float("inf")):
        x = t["x"].clone()
        x[17, 5] = bad
        for major in (False, True):
            got = slk.residual_norm(x, t["weight"], t["bias"], feature_major=major, **args)
            keep = [i for i in range(40) if i != 17]
            for a, b in zip(got, clean):
                torch.testing.assert_close(a[keep], b[keep], rtol=1e-5, atol=1e-6)
            assert bool(torch.isnan(got[1][17]).all())


def test_large_means_and_constant_rows(dev):
    x = torch.full((3, 384), 1e4, device=dev)
    x[1] += torch.randn(384, generator=torch.Generator().manual_seed(0)).to(dev)
    w, b = torch.ones(384, device=dev), torch.zeros(384, device=dev)
    y = slk.residual_norm(x, w, b)[1]
    want = F.layer_norm(x.double(), (384,), eps=1e-5)
    # the mean of values near 1e4 is off by a few 2^-24 · 1e4 = 6e-4; constant rows stay ~0
    # relative to 1/sqrt(eps) = 316 times that
    assert float((y[1].double() - want[1]).abs().max()) < 5e-3
    assert float(y[0].abs().max()) < 0.7


def test_empty_input(dev):
    w = torch.ones(64, device=dev, requires_grad=True)
    x = torch.zeros(0, 64, device=dev, requires_grad=True)
    u = torch.zeros(0, 64, device=dev, requires_grad=True)
    r, y = slk.residual_norm(x, w, branch=u)
    (r.sum() + y.sum()).backward()
    assert y.shape == (0, 64) and bool((w.grad == 0).all()) and x.grad.shape == (0, 64)


def test_between_two_sparse_layers_no_transposing_copy(dev, monkeypatch):
    torch.manual_seed(0)
    a = slk.SparseLinear(96, 128, sparsity=0.8, bias=False).to(dev)
    b = slk.SparseLinear(128, 80, sparsity=0.8, bias=False).to(dev)
    w = torch.ones(128, device=dev, requires_grad=True)
    x = torch.randn(4, 30, 96, device=dev)
    res = torch.randn(4, 30, 128, device=dev, requires_grad=True)
    u = a(x)
    copies = []
    real = _lib.transpose_dense
    monkeypatch.setattr(_lib, "transpose_dense", lambda s, d: (copies.append(s.shape), real(s, d)))
    r, y = slk.residual_norm(res, w, branch=u, feature_major=True)
    out = b(y)
    assert not copies
    grads = torch.autograd.grad(out, [res, w, *a.parameters()], out.detach().clone())
    assert not copies
    assert all(bool(torch.isfinite(g).all()) for g in grads)


def test_another_stream(dev):
    t, dr, dy = make((64,), 384, "layer", True, "element", torch.float32, dev)
    args = {k: v for k, v in t.items() if k not in ("x", "weight", "bias")}
    want = slk.residual_norm(t["x"], t["weight"], t["bias"], **args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = slk.residual_norm(t["x"], t["weight"], t["bias"], **args)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(dev):
    x, w = torch.zeros(4, 6, 32, device=dev), torch.ones(32, device=dev)
    f = slk.residual_norm
    with pytest.raises(TypeError):
        f([1.0], w)
    with pytest.raises(RuntimeError, match="HIP"):
        f(x.cpu(), w)
    with pytest.raises(RuntimeError, match="HIP"):
        f(x, w.cpu())
    for bad in (dict(kind="batch"), dict(gate=w), dict(post_weight=w), dict(branch=x[:2]),
                dict(branch=x.bfloat16()), dict(branch=x, gate=x[:, :1, :16]),
                dict(branch=x, gate=x[:, :3]), dict(branch=x, gate=x[0]),
                dict(branch=x, gate=x[:1]), dict(branch=x, post_bias=w),
                dict(branch=x, kind="rms", post_weight=w, post_bias=w)):
        with pytest.raises(ValueError):
            f(x, w, **bad)
    with pytest.raises(ValueError, match="bias"):
        f(x, w, w, kind="rms")
    with pytest.raises(ValueError, match="shape"):
        f(x, w[:31])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        f(x.half(), w.half())
    with pytest.raises(ValueError, match="features"):
        f(torch.zeros(2, 16385, device=dev), torch.zeros(16385, device=dev))
    two = x.reshape(24, 32)
    with pytest.raises(ValueError, match="gate"):
        f(two, w, branch=two, gate=two[:5])


def test_double_backward_is_refused(dev):
    t, _, _ = make((4,), 64, "layer", False, "none", torch.float32, dev)
    x = t["x"].requires_grad_()
    up = torch.ones(4, 64, device=dev, requires_grad=True)
    g, = torch.autograd.grad(slk.residual_norm(x, t["weight"], t["bias"])[1], x, up,
                             create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,gate_rows,cols", [(1, 1, 1, 0), (7, 100, 7, 0), (9, 1027, 3, 0),
                                                (50, 300, 2, 1), (33, 1024, 1, 1), (6, 9000, 2, 0),
                                                (600, 64, 30, 1), (5000, 68, 5, 0)])
def test_writes_stay_in_range(dev, dtype, n, d, gate_rows, cols):
    """Through the C-ABI with guard bytes around every array that it may write."""
    g = torch.Generator().manual_seed(0)
    size = torch.empty(0, dtype=dtype).element_size()

    def rand(*s):
        return torch.randn(*s, generator=g).to(dtype).to(dev)

    guards = []

    def out(nbytes):
        buf = torch.full((nbytes + 1024,), 0xA5, dtype=torch.uint8, device=dev)
        guards.append(buf)
        return buf.data_ptr() + 512

    keep = {k: rand(n, d) for k in ("x", "branch", "dr", "dy")}
    keep |= {k: rand(d) for k in ("weight", "bias", "post_weight", "post_bias")}
    keep["gate"] = rand(gate_rows, d)
    args = _lib.Norm(n=n, d=d, gate_rows=gate_rows, scale=0.5, eps=1e-5,
                     dtype=_lib.DTYPES[dtype], layer=1, branch_cols=cols, y_cols=cols,
                     **{k: v.data_ptr() for k, v in keep.items()})
    args.r, args.y, args.stats = out(size * n * d), out(size * n * d), out(16 * n)
    _lib.norm_forward(args, _lib.stream_of(keep["x"]))
    args.dx, args.dbranch = out(size * n * d), out(size * n * d)
    args.dgate = out(size * gate_rows * d)
    for k in ("dweight", "dbias", "dpost_weight", "dpost_bias"):
        setattr(args, k, out(size * d))
    args.workspace_bytes = _lib.norm_workspace_bytes(args)
    args.workspace = out(args.workspace_bytes)
    _lib.norm_backward(args, _lib.stream_of(keep["x"]))
    torch.cuda.synchronize()
    for b in guards:
        assert bool((b[:512] == 0xA5).all()) and bool((b[-512:] == 0xA5).all())


def test_captured_norm_replays(dev):
    t, dr, dy = make((2, 100), 96, "layer", True, "sequence", torch.float32, dev)
    for v in t.values():
        v.requires_grad_()
    args = {k: v for k, v in t.items() if k not in ("x", "weight", "bias")}

    def once():
        r, y = slk.residual_norm(t["x"], t["weight"], t["bias"], **args)
        return (r.detach(), y.detach(), *torch.autograd.grad([r, y], list(t.values()), [dr, dy]))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        got = once()
    assert "memset" not in _lib.graph_node_types(graph)
    graph.instantiate()
    for k in range(4):
        with torch.no_grad():
            t["x"].copy_(torch.randn(2, 100, 96, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, once()))
