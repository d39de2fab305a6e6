"""attention's results against their own sizes: long rows, and rows of sizes far apart.

Bounds. Long rows, float32, u = 2^-24: a log-sum below 16 is rounded by 8u of its weights, a
weight's exponent by as much, an operand in two parts by 4u, dS likewise: 16u in the root of
their squares. A result is summed by the matrix cores sixteen keys (queries) at a time in three
products, each sum rounded by u of what it has reached: sqrt(3 n / 16) u for n keys, as roundings
at random add up. Rows of different sizes are held against the bound of test_gpu_attention.py,
each against its own row's terms.
"""

from __future__ import annotations

import pytest
import torch

import sparsecore_amd as slk
from test_gpu_attention import BF16, F32, Ref, close, feature_major, make

pytestmark = pytest.mark.gpu


def errors(got, want):
    """Of the whole, and of each row."""
    got, want = got.detach().double().cpu().reshape(want.shape), want
    off = got - want
    return float(off.norm() / want.norm()), off.norm(dim=-1) / want.norm(dim=-1)


def bound(n):
    return ((3 * n / 16) ** 0.5 + 16) * 2.0 ** -24


@pytest.mark.parametrize("tq,tk", [(64, 4096), (64, 8192), (40, 32768), (8192, 64), (1500, 1500)])
@pytest.mark.parametrize("d", [64, 128])
def test_float32_gradients_at_length(dev, tq, tk, d):
    q, k, v, do = make((1, tq), (1, tk), 1, 1, d, F32, dev)
    ref = Ref(q, k, v, do, [(0, tq, 0, tk)], False, d ** -0.5)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = slk.attention(*leaves, causal=False)
    for name, x, n in zip(("out", "dq", "dk", "dv"),
                          (out, *torch.autograd.grad(out, leaves, do)), (tk, tk, tq, tq)):
        whole, _ = errors(x, ref.val[name])
        assert whole <= bound(n), (name, whole, bound(n))


@pytest.mark.parametrize("tk", [512, 8192])
def test_one_large_gradient_among_small_ones(dev, tk):
    """A row of dO a thousand times its neighbours: their gradients are as exact as without."""
    q, k, v, do = make((1, 64), (1, tk), 1, 1, 64, F32, dev)
    do[0, 5] *= 1000
    ref = Ref(q, k, v, do, [(0, 64, 0, tk)], False, 0.125)
    q.requires_grad_()
    dq, = torch.autograd.grad(slk.attention(q, k, v, causal=False), [q], do)
    _, rows = errors(dq, ref.val["dq"])
    assert float(rows.median()) <= bound(tk), (float(rows.median()), bound(tk))


def rows_close(name, got, ref, dtype):
    """test_gpu_attention's bound with each row's own terms in place of all rows'."""
    want, mag = ref.val[name], ref.mag[name]
    got = got.detach().double().cpu().reshape(want.shape)
    share = 1e-5 if dtype is F32 else 2.0 ** (-7 if name in ("out", "dv") else -6)
    row = mag.square().mean(-1, keepdim=True).sqrt()
    off = (got - want).abs() - share * (mag + 1e-3 * row)
    assert not got.isnan().any(), name
    worst = int(off.flatten().argmax())
    assert float(off.max()) <= 1e-37, (name, worst, float(got.flatten()[worst]),
                                       float(want.flatten()[worst]), float(mag.flatten()[worst]))


def by_tiles(x, factors):
    """Rows 64 i .. 64 i + 63 times factors[i]."""
    t = x.shape[1]
    f = torch.tensor([factors[min(i // 64, len(factors) - 1)] for i in range(t)],
                     dtype=torch.float64)
    return (x.double().cpu() * f[None, :, None, None]).to(x.dtype).to(x.device)


SIZES = [[2.0 ** (20 * i) for i in range(5)], [2.0 ** (-20 * i) for i in range(5)],
         [1.0, 2.0 ** 40, 1.0, 2.0 ** -40, 1.0], [1.0, 1.0, 1.0, 1.0, 2.0 ** 90]]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("which", ["dout", "k"])
@pytest.mark.parametrize("d,buckets", [(64, 0), (128, 0), (32, 16)])
def test_gradients_of_tiles_of_different_sizes(dev, d, buckets, which, sizes, dtype):
    """dO or K over many powers of two from one 64 rows to the next of a causal sequence. (K so
    small that no score reaches a thousand.) What a row does not see is in none of its sums."""
    t, h = 300, 2
    q, k, v, do = make((1, t), (1, t), h, 1, d, dtype, dev)
    if which == "dout":
        do = by_tiles(do, sizes)
    else:
        top = max(sizes)
        k = by_tiles(k, [x / top for x in sizes])
    bias = torch.randn(buckets, h, device=dev) if buckets else None
    ref = Ref(q, k, v, do, [(0, t, 0, t)], True, d ** -0.5, bias, 20)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = slk.attention(*leaves, bias=bias, max_distance=20)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do))):
        rows_close(name, x, ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,buckets,t", [(64, 0, 300), (128, 0, 300), (32, 16, 300), (64, 0, 70)])
def test_values_of_tiles_of_different_sizes(dev, d, buckets, t, causal, sizes, dtype):
    """V over many powers of two from one 64 rows to the next: outputs and gradients, with and
    without what a backward keeps."""
    h = 2
    q, k, v, do = make((1, t), (1, t), h, 1, d, dtype, dev)
    v = by_tiles(v, sizes)
    bias = torch.randn(buckets, h, device=dev) if buckets else None
    ref = Ref(q, k, v, do, [(0, t, 0, t)], causal, d ** -0.5, bias, 20)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = slk.attention(*leaves, bias=bias, max_distance=20, causal=causal)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do))):
        rows_close(name, x, ref, dtype)
    with torch.no_grad():
        rows_close("out", slk.attention(q, k, v, bias=bias, max_distance=20, causal=causal),
                   ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("s,size", [(70, 2.0 ** 60), (3000, 2.0 ** 60), (3000, 2.0 ** -60)])
def test_values_that_hardly_count(dev, s, size, dtype):
    """A tile of values of another size that all queries give weights of about 2^-70: where
    these are large they still count, and where they are small nothing else is lost."""
    t, h, d = 40, 1, 64
    q, k, v, do = make((1, t), (1, s), h, h, d, dtype, dev)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, :64, :, 0] = -48.0  # scores of these keys lower by 48, about 2^-70 of the others' weight
    v[:, :64] *= size
    ref = Ref(q, k, v, do, [(0, t, 0, s)], False, 0.125)
    with torch.no_grad():
        rows_close("out", slk.attention(q, k, v, causal=False), ref, dtype)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = slk.attention(*leaves, causal=False)
    rows_close("out", out, ref, dtype)
    dq, = torch.autograd.grad(out, [leaves[0]], do)
    rows_close("dq", dq, ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_values_hidden_by_a_bias(dev, dtype):
    """Far keys, behind a bias of the lowest value, with values of 2^60."""
    t, h, d = 400, 2, 64
    q, k, v, do = make((1, t), (1, t), h, h, d, dtype, dev)
    v[:, :192] *= 2.0 ** 60
    bias = torch.randn(8, h, device=dev)
    bias[-1] = torch.finfo(F32).min
    ref = Ref(q, k, v, do, [(0, t, 0, t)], True, d ** -0.5, bias.clamp(min=-1e30), 40)
    out = slk.attention(q, k, v, bias=bias, max_distance=40)
    got, want = out.double().cpu().reshape(ref.val["out"].shape), ref.val["out"]
    rows = (got - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(rows.max()) <= (1e-5 if dtype is F32 else 2.0 ** -7)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", SIZES[:3])
def test_values_of_different_sizes_behind_lowest_biases(dev, sizes, dtype):
    """All biases of the lowest value: each output is the plain mean of the values it sees."""
    t, h, d = 300, 2, 64
    q, k, v, do = make((1, t), (1, t), h, h, d, dtype, dev)
    v = by_tiles(v, sizes)
    ref = Ref(torch.zeros_like(q), k, v, do, [(0, t, 0, t)], True, d ** -0.5)
    bias = torch.full((8, h), torch.finfo(F32).min, device=dev)
    rows_close("out", slk.attention(q, k, v, bias=bias, max_distance=20), ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [2.0 ** 30, 1e13, 1e30])
@pytest.mark.parametrize("at", [0, 63, 90, 149])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("d,buckets", [(64, 0), (128, 16), (32, 0), (40, 8)])
def test_one_row_much_larger_than_those_around_it(dev, d, buckets, which, at, size, dtype):
    """What does not see the row, or is not seen by it, is as exact as without it; what does is
    exact for its own size. (A large key or query: zeros but for a feature that all queries, or
    keys, have a zero in, so that no score grows.)"""
    t, h, g = 150, 2, 1
    q, k, v, do = make((1, t), (1, t), h, g, d, dtype, dev)
    q[..., 0], k[..., 0] = 0.0, 0.0
    x = {"q": q, "k": k, "v": v, "dout": do}[which]
    if which in "qk":
        x[0, at], x[0, at, :, 0] = 0.0, size
    else:
        x[0, at] *= size
    bias = torch.randn(buckets, h, device=dev).requires_grad_() if buckets else None
    ref = Ref(q, k, v, do, [(0, t, 0, t)], True, d ** -0.5, bias, 20)
    leaves = [y.requires_grad_() for y in (q, k, v)]
    out = slk.attention(*leaves, bias=bias, max_distance=20)
    grads = torch.autograd.grad(out, leaves + ([bias] if buckets else []), do)
    for name, y in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        rows_close(name, y, ref, dtype)
    if buckets:
        close("dbias", grads[3], ref, dtype)
    with torch.no_grad():
        rows_close("out", slk.attention(q, k, v, bias=bias, max_distance=20), ref, dtype)


def uneven(x, lo, hi, seed):
    """Every row times a power of two of its own."""
    gen = torch.Generator().manual_seed(seed)
    e = torch.randint(lo, hi + 1, x.shape[:-2], generator=gen).double()
    return (x.double().cpu() * (2.0 ** e)[..., None, None]).to(x.dtype).to(x.device)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,g,d,buckets", [(4, 2, 64, 0), (4, 1, 128, 0), (2, 2, 32, 16),
                                           (3, 3, 128, 16), (4, 2, 50, 0)])
def test_rows_of_all_sizes_in_packed_sequences(dev, h, g, d, buckets, causal, cols, dtype):
    lens = [1, 130, 0, 64, 65, 300]
    n = sum(lens) + 3
    q, k, v, do = make((n,), (n,), h, g, d, dtype, dev)
    q, k = uneven(q, -30, 0, 1), uneven(k, -30, 0, 2)
    v, do = uneven(v, -30, 30, 3), uneven(do, -30, 30, 4)
    if cols:
        q, k, v, do = (feature_major(x, (n,)) for x in (q, k, v, do))
    bias = torch.randn(buckets, h, device=dev) if buckets else None
    off = torch.tensor([0] + lens).cumsum(0)
    seqs = [(int(a), m, int(a), m) for a, m in zip(off, lens)]
    ref = Ref(q, k, v, do, seqs, causal, d ** -0.5, bias)
    more = {"offsets": off.int().to(dev), "causal": causal, "bias": bias, "feature_major": cols}
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = slk.attention(*leaves, **more)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do))):
        rows_close(name, x, ref, dtype)
    with torch.no_grad():
        rows_close("out", slk.attention(q, k, v, **more), ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("buckets", [0, 16])
def test_rows_of_all_sizes_in_split_keys(dev, buckets, dtype):
    b, t, s, h, d = 2, 70, 3001, 2, 64
    q, k, v, do = make((b, t), (b, s), h, 1, d, dtype, dev)
    k, v = uneven(k, -30, 0, 2), uneven(v, -30, 30, 3)
    bias = torch.randn(buckets, h, device=dev) if buckets else None
    ref = Ref(q, k, v, do, [(i * t, t, i * s, s) for i in range(b)], True, d ** -0.5, bias)
    with torch.no_grad():
        rows_close("out", slk.attention(q, k, v, bias=bias), ref, dtype)


def test_uneven_and_even_calls_in_one_graph(dev):
    """A captured step replayed with even rows, uneven ones and even ones again."""
    t, h, d = 300, 2, 64
    q, k, v, do = make((1, t), (1, t), h, 1, d, F32, dev)
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def step(*x):
        out = slk.attention(*x)
        return [out.detach(), *torch.autograd.grad(out, x, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*leaves)
    for i in range(4):
        new = make((1, t), (1, t), h, 1, d, F32, dev, seed=i + 1)
        with torch.no_grad():
            for x, y in zip((q, k, v, do), new):
                x.copy_(uneven(y, -30, 0, i) if i % 2 else y)
        graph.replay()
        torch.cuda.synchronize()
        seen = [x.clone() for x in got]
        want = step(*(x.detach().clone().requires_grad_() for x in leaves))
        assert all(torch.equal(a, b) for a, b in zip(seen, want)), i
        ref = Ref(q, k, v, do, [(0, t, 0, t)], True, d ** -0.5)
        for name, x in zip(("out", "dq", "dk", "dv"), seen):
            rows_close(name, x, ref, F32)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b,t,h,g,d,buckets", [(200, 4, 2, 1, 64, 0), (100, 9, 2, 2, 128, 0),
                                               (100, 7, 2, 2, 32, 8), (3, 150, 4, 2, 64, 0),
                                               (2, 300, 2, 1, 128, 16)])
def test_bfloat16_is_rounded_to_11_bits_between_the_products(dev, b, t, h, g, d, buckets, causal):
    """A result is rounded to bfloat16, half a step: 2^-8 of it. A weight, or dS, is rounded to
    float16: 2^-11 of each term. O as it is read by the backward is off by 2^-8 of 2^-8 of it,
    scores and sums by what float32 has (1e-5 of a term, see test_gpu_attention.py): 2^-14 of
    each term covers both. (Weights or O in bfloat16 would be off by 2^-8 of the terms.)"""
    q, k, v, do = make((b, t), (b, t), h, g, d, BF16, dev)
    bias = torch.randn(buckets, h, device=dev) if buckets else None
    ref = Ref(q, k, v, do, [(i * t, t, i * t, t) for i in range(b)], causal, d ** -0.5, bias)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = slk.attention(*leaves, causal=causal, bias=bias)
    half = torch.finfo(BF16).eps / 2
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do))):
        want, mag = ref.val[name], ref.mag[name]
        got = x.detach().double().cpu().reshape(want.shape)
        off = (got - want).abs() - half * want.abs() - (2.0 ** -11 + 2.0 ** -14) * mag
        assert float(off.max()) <= 0, (name, float(off.max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("least", [-10, -12, -14, -16])
def test_rows_about_as_far_apart_as_one_power_of_two_serves(dev, least, dtype):
    """On both sides of the spread from which rows have exponents of their own."""
    t, h, d = 300, 2, 64
    q, k, v, do = make((1, t), (1, t), h, 1, d, dtype, dev)
    q, k = uneven(q, least, 0, 1), uneven(k, least, 0, 2)
    v, do = uneven(v, least, 0, 3), uneven(do, least, 0, 4)
    ref = Ref(q, k, v, do, [(0, t, 0, t)], True, d ** -0.5)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = slk.attention(*leaves)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do))):
        rows_close(name, x, ref, dtype)
