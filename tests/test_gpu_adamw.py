"""AdamW over many tensors (slk_adamw), 8-bit moments (slk_q8_*), moments that follow a
topology rewrite (slk_carry_slots), and the optimizer built on them.

The step is checked against the formula in float64. Bound of a float32 step, u = 2^-24:
m and v are two products and a sum each (v has the square too), the square root, its
scaling, the added eps, the quotient, the step size and two products and a difference
round once each, the constants (decay, step size, 1 / sqrt(1 - b2^t), 1 - b1, 1 - b2)
once; v enters through its root, which halves its relative error. With
M = b1 |m| + (1 - b1) |g| the update's error is below 14 u · step · M / root and that of
p below 3 u |p| more; m's is below 4 u M, v's 5 u v. Codes are compared exactly with the
same float32 operations in numpy, each of them correctly rounded on both sides.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import sparsecore_amd as slk
from sparsecore_amd import optim

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.98, 1e-8, 0.05
SIZES = [1, 3, 4, 255, 256, 257, 1023, 1024, 1025, 5000, 0, 70001]


def np_encode(x, signed):
    """(codes, scales) of a flat float32 array, operation by operation in float32."""
    f = np.float32
    blocks = -(-x.size // 256)
    pad = np.zeros(blocks * 256, f)
    pad[:x.size] = x
    pad = pad.reshape(blocks, 256)
    scale = np.abs(pad).max(axis=1).astype(f) if blocks else np.zeros(0, f)
    with np.errstate(all="ignore"):
        a = np.where(scale[:, None] > 0, np.abs(pad) / scale[:, None], f(0)).astype(f)
    if signed:
        q = np.rint(np.sqrt(a) * f(127))
        codes = np.copysign(q, pad).astype(np.int8)
    else:
        q = np.rint(np.sqrt(np.sqrt(a)) * f(255))
        codes = np.where(pad > 0, np.maximum(q, 1), q).astype(np.uint8)
    return codes.reshape(-1)[:x.size], scale


def np_decode(codes, scale):
    f = np.float32
    s = np.repeat(scale, 256)[:codes.size]
    if codes.dtype == np.int8:
        t = codes.astype(f) * f(1.0 / 127.0)
        return (t * np.abs(t)) * s
    t = codes.astype(f) * f(1.0 / 255.0)
    t = t * t
    return (t * t) * s


def tensors(sizes, dtype, seed, dev, offset=0):
    """(p, g, m, v) lists; `offset` elements into their buffers, for odd alignments."""
    g = torch.Generator().manual_seed(seed)

    def make(scale, dt, square=False):
        out = []
        for n in sizes:
            x = torch.randn(n + offset, generator=g) * scale
            x = x * torch.exp(2 * torch.randn(n + offset, generator=g))
            out.append((x.square() if square else x).to(dt).to(dev)[offset:])
        return out

    return (make(0.05, dtype), make(1e-3, dtype), make(3e-4, torch.float32),
            make(1e-3, torch.float32, square=True))


def reference(p, g, m, v, step):
    p, g, m, v = (t.double().cpu() for t in (p, g, m, v))
    M = B1 * m.abs() + (1 - B1) * g.abs()
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * g * g
    root = v.sqrt() / math.sqrt(1 - B2 ** step) + EPS
    size = LR / (1 - B1 ** step)
    want = (1 - LR * WD) * p - size * m / root
    return want, m, v, U * (3 * p.abs() + 14 * size * M / root), 4 * U * M, 5 * U * v


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("step", [1, 1000])
def test_step_matches_the_formula(dev, dtype, offset, step):
    p, g, m, v = tensors(SIZES, dtype, 1, dev, offset)
    want = [reference(*t, step) for t in zip(p, g, m, v)]
    optim.adamw_step(p, g, m, v, step=step, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    for i, n in enumerate(SIZES):
        wp, wm, wv, ep, em, ev = want[i]
        if dtype is torch.bfloat16:
            ep = ep + 2.0 ** -8 * (wp.abs() + ep) + 2.0 ** -133  # one rounding to 8 bits
        for got, w, e, what in ((p[i], wp, ep, "p"), (m[i], wm, em, "m"), (v[i], wv, ev, "v")):
            assert bool(((got.double().cpu() - w).abs() <= e + 1e-44).all()), (n, what)


def test_more_tensors_than_a_launch_holds_and_two_dtypes(dev):
    sizes = [(37 * i) % 600 for i in range(150)]
    kinds = [torch.bfloat16 if i % 3 == 0 else torch.float32 for i in range(150)]
    parts = [tensors([n], k, i, dev) for i, (n, k) in enumerate(zip(sizes, kinds))]
    p, g, m, v = ([t[j][0] for t in parts] for j in range(4))
    want = [reference(*t, 7) for t in zip(p, g, m, v)]
    optim.adamw_step(p, g, m, v, step=7, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    for i in range(150):
        wp, _, wv, ep, _, ev = want[i]
        if kinds[i] is torch.bfloat16:
            ep = ep + 2.0 ** -8 * (wp.abs() + ep) + 2.0 ** -133
        assert bool(((p[i].double().cpu() - wp).abs() <= ep + 1e-44).all()), i
        assert bool(((v[i].double().cpu() - wv).abs() <= ev + 1e-44).all()), i


def test_padding_slots_stay_zero_and_neighbours_untouched(dev):
    buf = torch.full((1000,), 7.0, device=dev)
    p, g = buf[100:400], torch.zeros(300, device=dev)
    p.zero_()
    m, v = torch.zeros(300, device=dev), torch.zeros(300, device=dev)
    optim.adamw_step([p], [g], [m], [v], step=1, lr=LR)
    assert bool((p == 0).all()) and bool((m == 0).all()) and bool((v == 0).all())
    assert bool((buf[:100] == 7).all()) and bool((buf[400:] == 7).all())


def test_step_and_lr_on_the_device_give_the_same_step(dev):
    a, b = tensors([1000], torch.float32, 2, dev), tensors([1000], torch.float32, 2, dev)
    optim.adamw_step(*a, step=12, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    optim.adamw_step(*b, step=torch.tensor([12.0], device=dev), lr=torch.tensor([LR], device=dev),
                     betas=(B1, B2), eps=EPS, weight_decay=WD)
    # the learning rate is rounded to float32 once more, the coefficients differ by an ulp
    for x, y in zip(a, b):
        torch.testing.assert_close(x[0], y[0], rtol=1e-6, atol=1e-9)


# ───────────────────────── 8-bit moments ─────────────────────────

@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("n", [1, 255, 256, 257, 4096, 70001])
def test_codes_are_the_maps(dev, signed, n):
    x = torch.randn(n, generator=torch.Generator().manual_seed(n)) * 1e-3
    x = x * torch.exp(3 * torch.randn(n, generator=torch.Generator().manual_seed(n + 1)))
    x[::7] = 0.0
    x = x if signed else x.abs()
    codes, scales = optim.quantize(x.to(dev), signed)
    wc, ws = np_encode(x.numpy(), signed)
    assert np.array_equal(codes.cpu().numpy(), wc) and np.array_equal(scales.cpu().numpy(), ws)
    back = optim.dequantize(codes, scales).cpu().numpy()
    assert np.array_equal(back, np_decode(wc, ws))
    # values that stand for themselves: encoding what was decoded changes no code
    again, s2 = optim.quantize(torch.from_numpy(back).to(dev), signed)
    assert torch.equal(again, codes) and torch.equal(s2, scales)


def test_zero_blocks_tiny_second_moments_and_non_finite_blocks(dev):
    x = torch.zeros(768)
    x[256] = 1.0
    x[257] = 1e-30  # far below a step: code 1, not 0
    codes, scales = optim.quantize(x.to(dev), False)
    assert codes[:256].sum() == 0 and scales[0] == 0 and scales[2] == 0
    assert int(codes[256]) == 255 and int(codes[257]) == 1 and codes[258:].sum() == 0
    for bad in (math.inf, math.nan):
        x = torch.randn(768, generator=torch.Generator().manual_seed(1)).abs()
        x[300] = bad
        for signed in (True, False):
            got = optim.dequantize(*optim.quantize(x.to(dev), signed)).cpu()
            assert bool(torch.isnan(got[256:512]).all())
            assert bool(torch.isfinite(got[:256]).all() and torch.isfinite(got[512:]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 3])
def test_8bit_step_is_the_32bit_step_on_the_decoded_moments(dev, dtype, offset):
    p, g, m, v = tensors(SIZES, dtype, 5, dev)
    (mc, ms), (vc, vs) = (zip(*[optim.quantize(x, signed) for x in t])
                          for t, signed in ((m, True), (v, False)))

    def shifted(codes):  # the same codes at an odd address
        out = []
        for c in codes:
            buf = torch.zeros(c.numel() + offset, dtype=c.dtype, device=dev)
            buf[offset:] = c
            out.append(buf[offset:])
        return out

    mc, vc, ms, vs = shifted(mc), shifted(vc), list(ms), list(vs)
    m32 = [optim.dequantize(c.clone(), s) for c, s in zip(mc, ms)]
    v32 = [optim.dequantize(c.clone(), s) for c, s in zip(vc, vs)]
    p32 = [x.clone() for x in p]
    optim.adamw_step(p32, g, m32, v32, step=9, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    optim.adamw_step(p, g, mc, vc, exp_avg_scales=ms, exp_avg_sq_scales=vs, step=9, lr=LR,
                     betas=(B1, B2), eps=EPS, weight_decay=WD)
    for i in range(len(SIZES)):
        assert torch.equal(p[i], p32[i]), SIZES[i]
        for codes, scales, full, signed in ((mc, ms, m32, True), (vc, vs, v32, False)):
            wc, ws = np_encode(full[i].cpu().numpy(), signed)
            assert np.array_equal(codes[i].cpu().numpy(), wc)
            assert np.array_equal(scales[i].cpu().numpy(), ws)


# ───────────────────────── moments that follow ─────────────────────────

def topologies(rows, cols, seed, empty=False):
    """(row_start, old, new) numpy arrays: random rows before and after, of any lengths up
    to their capacities."""
    rng = np.random.default_rng(seed)
    cap = rng.integers(1, cols + 1, rows)
    start = np.concatenate([[0], np.cumsum(cap)[:-1]]).astype(np.int32)
    out = []
    for _ in range(2):
        nnz = np.array([rng.integers(0, c + 1) for c in cap], dtype=np.int32)
        if empty:
            nnz[::2] = 0
        at = np.full(int(cap.sum()), -1, dtype=np.int32)
        for r in range(rows):
            at[start[r]:start[r] + nnz[r]] = np.sort(rng.choice(cols, nnz[r], replace=False))
        out.append((at, nnz))
    return start, out[0], out[1]


def moved(start, old, new, x):
    out = np.zeros_like(x)
    for r in range(len(start)):
        was = {int(old[0][s]): s for s in range(start[r], start[r] + old[1][r])}
        for s in range(start[r], start[r] + new[1][r]):
            if int(new[0][s]) in was:
                out[s] = x[was[int(new[0][s])]]
    return out


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 1000), (300, 1), (7, 300), (513, 40)])
@pytest.mark.parametrize("empty", [False, True])
def test_carried_states_are_their_slots(dev, rows, cols, empty):
    start, old, new = topologies(rows, cols, rows + cols, empty)
    total = old[0].size
    rng = np.random.default_rng(1)
    m = rng.standard_normal(total).astype(np.float32)
    v = (m * m).astype(np.float32)
    t = [torch.from_numpy(a).to(dev) for a in (start, *old, *new)]
    (mc, ms), (vc, vs) = np_encode(m, True), np_encode(v, False)
    states = [torch.from_numpy(m).to(dev), torch.from_numpy(v).to(dev),
              (torch.from_numpy(mc).to(dev), torch.from_numpy(ms).to(dev)),
              (torch.from_numpy(vc).to(dev), torch.from_numpy(vs).to(dev))]
    got = optim.carry_slots(t[0], (t[1], t[2]), (t[3], t[4]), states)
    assert np.array_equal(got[0].cpu().numpy(), moved(start, old, new, m))
    assert np.array_equal(got[1].cpu().numpy(), moved(start, old, new, v))
    for k, codes, scales, signed in ((2, mc, ms, True), (3, vc, vs, False)):
        wc, ws = np_encode(moved(start, old, new, np_decode(codes, scales)), signed)
        assert np.array_equal(got[k][0].cpu().numpy(), wc)
        assert np.array_equal(got[k][1].cpu().numpy(), ws)


# ───────────────────────── the optimizer ─────────────────────────

def model(dev, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(slk.SparseLinear(64, 96, sparsity=0.8), torch.nn.ReLU(),
                               slk.SparseLinear(96, 80, sparsity=0.7, bias=False)).to(dev)


def backward(net, x):
    net.zero_grad(set_to_none=True)
    loss = net(x).square().mean()
    loss.backward()
    return loss.detach()


def test_optimizer_follows_torchs_trajectory(dev):
    a, b = model(dev), model(dev)
    ours = slk.AdamW(a.parameters(), lr=1e-2, betas=(B1, B2), weight_decay=WD)
    theirs = torch.optim.AdamW(b.parameters(), lr=1e-2, betas=(B1, B2), weight_decay=WD)
    x = torch.randn(32, 64, generator=torch.Generator().manual_seed(3)).to(dev)
    for _ in range(5):
        backward(a, x), backward(b, x)
        # equal gradients: Adam's sign-like first steps would turn rounding into lr-sized steps
        for p, q in zip(a.parameters(), b.parameters()):
            q.grad.copy_(p.grad)
        ours.step(), theirs.step()
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p, q, rtol=2e-5, atol=2e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_follow_a_set_update(dev, bits):
    net = model(dev)
    opt = slk.AdamW(net.parameters(), lr=1e-2, state_bits=bits)
    net.apply(opt.attach)
    algo = slk.SET(sparsity=0.8, drop_fraction=0.3, update_freq=1, seed=1)
    net.apply(algo)
    x = torch.randn(32, 64, generator=torch.Generator().manual_seed(3)).to(dev)
    for _ in range(3):
        backward(net, x)
        opt.step()
        layer = net[0]
        csr, p = layer._csr, layer._values
        start = csr.row_start.cpu().numpy()
        old = csr.col_indices.cpu().numpy().copy(), csr.row_nnz.cpu().numpy().copy()
        s = opt.state[p]
        m = (optim.dequantize(s["exp_avg"], s["exp_avg_scale"]) if bits == 8
             else s["exp_avg"]).cpu().numpy().copy()
        algo.step()
        new = csr.col_indices.cpu().numpy(), csr.row_nnz.cpu().numpy()
        assert not np.array_equal(old[0], new[0])
        want = moved(start, old, new, m)
        if bits == 8:
            want = np_decode(*np_encode(want, True))
        net.zero_grad(set_to_none=True)
        p.grad = torch.zeros_like(p)  # a zero gradient leaves m = b1 · (the moved moment)
        opt.step()
        got = opt.state[p]["exp_avg"]
        if bits == 8:
            want = np_encode(np.float32(0.9) * want, True)
            assert np.array_equal(got.cpu().numpy(), want[0])
        else:
            assert np.array_equal(got.cpu().numpy(), np.float32(0.9) * want)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip_keeps_states_as_they_are(dev, bits):
    p = torch.nn.Parameter(torch.randn(700, device=dev).to(torch.bfloat16))
    opt = slk.AdamW([p], lr=1e-2, state_bits=bits)
    g = torch.randn(700, device=dev).to(torch.bfloat16)
    for _ in range(3):
        p.grad = g
        opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    twin = slk.AdamW([q], lr=1e-2, state_bits=bits)
    twin.load_state_dict(opt.state_dict())
    for k, v in opt.state[p].items():
        w = twin.state[q][k]
        assert (torch.equal(v, w) and v.dtype == w.dtype) if isinstance(v, torch.Tensor) else v == w
    p.grad = q.grad = g
    opt.step(), twin.step()
    assert torch.equal(p, q)


def test_captured_steps_count_their_replays(dev):
    a = [torch.nn.Parameter(torch.randn(n, device=dev)) for n in (1000, 37)]
    b = [torch.nn.Parameter(t.detach().clone()) for t in a]
    grads = [torch.randn_like(t) for t in a]
    eager = slk.AdamW(a, lr=1e-2)
    graphed = slk.AdamW(b, lr=1e-2, capturable=True)
    for p, q, g in zip(a, b, grads):
        p.grad, q.grad = g.clone(), g.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graphed.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.step()
    eager.step()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        for p, q in zip(a, b):
            torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-7)
    plain = slk.AdamW(a, lr=1e-2)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(graph):
            plain.step()


def test_late_gradients_begin_their_own_count(dev):
    for capturable in (False, True):
        a, b = (torch.nn.Parameter(torch.ones(10, device=dev)) for _ in range(2))
        opt = slk.AdamW([a, b], lr=1e-2, weight_decay=0.0, capturable=capturable)
        a.grad = torch.ones_like(a)
        opt.step()
        b.grad = torch.ones_like(b)
        opt.step()
        assert float(opt.state[a]["step"]) == 2 and float(opt.state[b]["step"]) == 1
        # a constant gradient: every bias-corrected step is lr
        torch.testing.assert_close(a, torch.full_like(a, 0.98), rtol=1e-6, atol=0)
        torch.testing.assert_close(b, torch.full_like(b, 0.99), rtol=1e-6, atol=0)


def test_a_replaced_matrix_is_refused(dev):
    net = model(dev)
    opt = slk.AdamW(net.parameters(), lr=1e-2)
    net.apply(opt.attach)
    x = torch.randn(32, 64, generator=torch.Generator().manual_seed(3)).to(dev)
    backward(net, x)
    opt.step()
    net.load_state_dict({k: v.clone() for k, v in net.state_dict().items()})
    backward(net, x)
    with pytest.raises(RuntimeError, match="attach"):
        opt.step()
    net.apply(opt.attach)
    opt.step()


def test_refusals(dev):
    p, g, m, v = tensors([10], torch.float32, 1, dev)
    kw = dict(step=1, lr=LR)
    for bad in (dict(step=0), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8),
                dict(weight_decay=-0.1), dict(step=torch.ones(2, device=dev))):
        with pytest.raises(ValueError):
            optim.adamw_step(p, g, m, v, **{**kw, **bad})
    with pytest.raises(ValueError, match="same length"):
        optim.adamw_step(p, g, m, [], **kw)
    with pytest.raises(ValueError, match="sizes"):
        optim.adamw_step(p, [g[0][:5]], m, v, **kw)
    with pytest.raises(ValueError, match="dtype"):
        optim.adamw_step(p, [g[0].bfloat16()], m, v, **kw)
    with pytest.raises(ValueError, match="moments"):
        optim.adamw_step(p, g, [m[0].bfloat16()], v, **kw)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        optim.adamw_step([p[0].half()], [g[0].half()], m, v, **kw)
    with pytest.raises(ValueError, match="contiguous"):
        big = torch.zeros(20, device=dev)
        optim.adamw_step([big[::2]], g, m, v, **kw)
    with pytest.raises(RuntimeError, match="HIP"):
        optim.adamw_step([p[0].cpu()], g, m, v, **kw)
    with pytest.raises(TypeError):
        optim.adamw_step([None], g, m, v, **kw)
    codes, scales = optim.quantize(m[0], True)
    sq, sq_scales = optim.quantize(v[0], False)
    with pytest.raises(ValueError, match="scales of both"):
        optim.adamw_step(p, g, [codes], [sq], exp_avg_scales=[scales], **kw)
    with pytest.raises(ValueError, match="scale per"):
        optim.adamw_step(p, g, [codes], [sq], exp_avg_scales=[scales],
                         exp_avg_sq_scales=[torch.zeros(2, device=dev)], **kw)
    with pytest.raises(ValueError, match="state_bits"):
        slk.AdamW([torch.nn.Parameter(p[0])], state_bits=16)
    with pytest.raises(ValueError, match="int8"):
        optim.dequantize(m[0], scales)
    with pytest.raises(ValueError, match="scales"):
        optim.dequantize(codes, scales[:0])
    start = torch.zeros(1, dtype=torch.int32, device=dev)
    cols = torch.arange(10, dtype=torch.int32, device=dev)
    nnz = torch.full((1,), 10, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="int32"):
        optim.carry_slots(start.long(), (cols, nnz), (cols, nnz), [m[0]])
    with pytest.raises(ValueError, match="same rows"):
        optim.carry_slots(start, (cols, nnz), (cols[:5], nnz), [m[0]])
    with pytest.raises(ValueError, match="per slot"):
        optim.carry_slots(start, (cols, nnz), (cols, nnz), [m[0][:5]])
    with pytest.raises(ValueError, match="at most"):
        optim.carry_slots(start, (cols, nnz), (cols, nnz), [m[0]] * 5)
    with pytest.raises(RuntimeError, match="HIP"):
        optim.carry_slots(start, (cols.cpu(), nnz), (cols, nnz), [m[0]])


@pytest.mark.parametrize("seed", range(4))
def test_carried_states_of_long_rows_that_shift_far(dev, seed):
    """Rows far longer than the slots around a place that the kernel looks at first:
    columns that stay, shift by a few slots, by hundreds (a block of columns dropped at
    one end and grown at the other) or by the whole row; rows of one slot between them."""
    rng = np.random.default_rng(seed)
    cols = 6000
    rows_old, rows_new, cap = [], [], []
    for _ in range(40):
        n = int(rng.choice([1, 3, 700, 2500, 5000]))
        a = np.sort(rng.choice(cols, n, replace=False))
        how = rng.integers(0, 4)
        keep = a[rng.random(n) > 0.3] if how == 0 else a[n // 3:] if how == 1 \
            else a[: n - n // 3] if how == 2 else a[:0]
        free = np.setdiff1d(np.arange(cols), a)
        grow = rng.choice(free, min(n - keep.size, free.size), replace=False)
        if how == 1:
            grow = np.sort(free)[-(n - keep.size):] if n > keep.size else free[:0]
        elif how == 2:
            grow = np.sort(free)[: n - keep.size]
        b = np.sort(np.concatenate([keep, grow]))
        rows_old.append(a), rows_new.append(b), cap.append(max(n, b.size) + int(rng.integers(1, 9)))
    start = np.concatenate([[0], np.cumsum(cap)[:-1]]).astype(np.int32)
    total = int(np.sum(cap))
    out = []
    for rows in (rows_old, rows_new):
        at, nnz = np.full(total, -1, np.int32), np.array([r.size for r in rows], np.int32)
        for s, r in zip(start, rows):
            at[s:s + r.size] = r
        out.append((at, nnz))
    old, new = out
    m = rng.standard_normal(total).astype(np.float32)
    t = [torch.from_numpy(x).to(dev) for x in (start, *old, *new, m)]
    got, = optim.carry_slots(t[0], (t[1], t[2]), (t[3], t[4]), [t[5]])
    assert np.array_equal(got.cpu().numpy(), moved(start, old, new, m))
