"""attention against its definition in float64, with the formulas' gradients, and its
gradients against differences.

Bounds. A result is a sum of terms, each a product of factors that carry errors of their
own, so errors are measured against the terms' absolute values (`Ref.mag`):

  out    sum_j p |v|,      dv  sum_i p |do|,
  ds     p (|do|·|v| + |do|·|out|) per pair, dq, dk: its sum times scale |k|, |q|; dbias: its sum

float32, u = 2^-24: an operand in two parts is off by 4u, a product of two with the dropped
lo·lo by 12u, a sum of 128 of them in any order by at most 128u more: 140u of
sum |q||k| for a score, which changes its weight by that share of A = scale sum |q||k| + |bias|.
The weights' own rounding, the exponential and the sums over keys add less than 28u, as long
as their roundings do not all point one way: 168u = 1e-5 of (1 + A)·mag covers both.
bfloat16, h = finfo.eps / 2 = 2^-8 (half a step): scores are float32; a weight is rounded to
bfloat16 (h of its terms), the result too (h): 2h = 2^-7 for out and dv. ds takes out rounded
by the forward (h), is rounded itself (h) and summed into a result that is (h): 3h, and
4h = 2^-6 leaves room for the float32 part, 1e-5 (1 + A).
"""

from __future__ import annotations

import pytest
import torch

import sparsecore_amd as slk
from sparsecore_amd.attn import relative_buckets

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def bucket_table(buckets, causal, md):
    """Bucket of each distance -md..md, from logarithms in float64 away from borders and
    whole numbers on them."""
    import math

    one = buckets if causal else buckets // 2
    e = one // 2
    out = []
    for d in range(-md, md + 1):
        n = abs(d)
        if n < e:
            b = n
        else:
            x = math.log(n / e) / math.log(md / e) * (one - e)
            t = round(x) if abs(x - round(x)) < 1e-9 else math.floor(x)
            b = min(one - 1, e + t)
        out.append(b if causal or d >= 0 else b + one)
    return torch.tensor(out)


class Ref:
    """out, gradients and their magnitudes in float64 on the CPU; sequences are
    (first query, queries, first key, keys) of row-flattened tensors."""

    def __init__(self, q, k, v, dout, seqs, causal, scale, bias=None, md=128):
        q, k, v, do = (x.detach().double().cpu().flatten(0, -3) for x in (q, k, v, dout))
        h, g = q.shape[1], k.shape[1]
        rep = h // g
        self.val = {n: torch.zeros_like(x) for n, x in
                    (("out", q), ("dq", q), ("dk", k), ("dv", v))}
        self.mag = {n: torch.zeros_like(x) for n, x in self.val.items()}
        b = bias.detach().double().cpu() if bias is not None else None
        if b is not None:
            self.val["dbias"], self.mag["dbias"] = torch.zeros_like(b), torch.zeros_like(b)
            near = bucket_table(b.shape[0], causal, md)
        for q0, nq, k0, nk in seqs:
            if nq == 0 or nk == 0:
                continue
            away = torch.arange(nq)[:, None] + (nk - nq) - torch.arange(nk)
            see = away >= 0 if causal else torch.ones(nq, nk, dtype=torch.bool)
            which = near[away.clamp(-md, md) + md] if b is not None else None
            for i in range(h):
                j = i // rep
                Q, K, V, G = q[q0:q0 + nq, i], k[k0:k0 + nk, j], v[k0:k0 + nk, j], \
                    do[q0:q0 + nq, i]
                # masked keys may hold anything
                s = torch.where(see, (Q @ K.t()) * scale, 0.0)
                a = torch.where(see, (Q.abs() @ K.abs().t()) * scale, 0.0)
                if b is not None:
                    s, a = s + b[which, i], a + b[which, i].abs()
                s = s.masked_fill(~see, -float("inf"))
                top = s.amax(1, keepdim=True)
                p = torch.exp(s - torch.where(top > -float("inf"), top, 0.0))
                total = p.sum(1, keepdim=True)
                p = torch.where(total > 0, p / total, 0.0)
                amp = 1 + torch.where(see, a, 0.0).amax(1, keepdim=True)
                o = p @ V
                dp, dpm = G @ V.t(), G.abs() @ V.abs().t()
                dl, dlm = (G * o).sum(1, keepdim=True), (G * o).abs().sum(1, keepdim=True)
                ds, dsm = p * (dp - dl), p * (dpm + dlm)
                add = {"out": (o, amp * (p @ V.abs()), q0, nq, i),
                       "dq": (scale * ds @ K, scale * (amp * dsm) @ K.abs(), q0, nq, i),
                       "dk": (scale * ds.t() @ Q, scale * (amp * dsm).t() @ Q.abs(), k0, nk, j),
                       "dv": (p.t() @ G, (amp * p).t() @ G.abs(), k0, nk, j)}
                for n, (x, m, r, rows, head) in add.items():
                    self.val[n][r:r + rows, head] += x
                    self.mag[n][r:r + rows, head] += m
                if b is not None:
                    for t, x in ((self.val, ds), (self.mag, amp * dsm)):
                        t["dbias"][:, i].index_add_(0, which.flatten(), x.flatten())


def close(name, got, ref, dtype):
    want, mag = ref.val[name], ref.mag[name]
    got = got.detach().double().cpu().reshape(want.shape)
    rms = mag.square().mean().sqrt()
    share = 1e-5 if dtype is F32 else 2.0 ** (-7 if name in ("out", "dv") else -6)
    off = (got - want).abs() - share * (mag + 1e-3 * rms)
    assert not got.isnan().any(), name
    assert float(off.max()) <= 0, (name, float(off.max()), float(rms),
                                   float((got - want).norm() / want.norm()))


def feature_major(x, lead):
    rows = x.reshape(-1, x.shape[-2] * x.shape[-1])
    return rows.t().contiguous().t().unflatten(1, x.shape[-2:]).unflatten(0, lead)


def make(lead_q, lead_k, h, g, d, dtype, dev, seed=0, layout="rows"):
    gen = torch.Generator().manual_seed(seed)

    def rand(*s, scale=1.0):
        return (scale * torch.randn(*s, generator=gen)).to(dtype).to(dev)

    q, k, v = rand(*lead_q, h, d, scale=1.3), rand(*lead_k, g, d, scale=1.3), rand(*lead_k, g, d)
    do = rand(*lead_q, h, d)
    if layout == "cols":
        q, do = feature_major(q, lead_q), feature_major(do, lead_q)
        k, v = feature_major(k, lead_k), feature_major(v, lead_k)
    elif layout == "qkv":  # slices of one projection's output
        both = torch.cat([x.flatten(-2) for x in (q, k, v)], -1)
        q, k, v = (x.unflatten(-1, (-1, d)) for x in both.split([h * d, g * d, g * d], -1))
    elif layout == "heads":  # (.., H, T, D) in memory
        q, k, v, do = (x.transpose(-2, -3).contiguous().transpose(-2, -3) for x in (q, k, v, do))
    return q, k, v, do


def check(dev, b, t, s, h, g, d, dtype, causal, layout="rows", buckets=0, md=128, scale=None,
          lengths=None, k_lengths=None, fm=False, seed=0):
    q, k, v, do = make((b, t), (b, s), h, g, d, dtype, dev, seed, layout)
    bias = None
    if buckets:
        gen = torch.Generator().manual_seed(seed + 1)
        bias = torch.randn(buckets, h, generator=gen).to(dev).requires_grad_()
    nq = lengths or [t] * b
    nk = k_lengths or lengths or [s] * b
    seqs = [(i * t, nq[i], i * s, nk[i]) for i in range(b)]
    ref = Ref(q, k, v, do, seqs, causal, scale if scale is not None else d ** -0.5, bias, md)
    for x in (q, k, v):
        x.requires_grad_()
    more = {n: torch.tensor(x, dtype=torch.int32, device=dev)
            for n, x in (("lengths", lengths), ("k_lengths", k_lengths)) if x}
    out = slk.attention(q, k, v, causal=causal, scale=scale, bias=bias, max_distance=md,
                        feature_major=fm, **more)
    assert out.shape == q.shape and out.dtype == dtype
    leaves = [q, k, v] + ([bias] if buckets else [])
    grads = torch.autograd.grad(out, leaves, do)
    for n, x in zip(("out", "dq", "dk", "dv", "dbias"), (out, *grads)):
        close(n, x, ref, dtype)
    for x, y in zip(grads, leaves):
        assert x.shape == y.shape and x.dtype == y.dtype
    with torch.no_grad():
        alone = slk.attention(q, k, v, causal=causal, scale=scale, bias=bias, max_distance=md,
                              feature_major=fm, **more)
    close("out", alone, ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("t,d,h,g", [(1, 64, 2, 2), (31, 64, 1, 1), (64, 32, 4, 2),
                                     (65, 128, 2, 1), (128, 64, 3, 3), (200, 40, 4, 1),
                                     (257, 80, 2, 2), (300, 128, 4, 2), (129, 1, 2, 1),
                                     (97, 33, 2, 2)])
def test_sizes(dev, t, d, h, g, dtype, causal):
    check(dev, 2, t, t, h, g, d, dtype, causal)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["cols", "qkv", "heads"])
@pytest.mark.parametrize("fm", [True, False])
def test_layouts(dev, layout, dtype, fm):
    check(dev, 2, 150, 150, 4, 2, 64, dtype, True, layout=layout, fm=fm)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("t,s", [(5, 200), (70, 300), (200, 70), (1, 129), (130, 1), (20, 64)])
def test_queries_and_keys_of_different_lengths(dev, t, s, dtype, causal):
    """With more queries than keys a causal mask leaves the first queries nothing."""
    check(dev, 2, t, s, 4, 2, 64, dtype, causal)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128, 24])
def test_bias(dev, d, dtype, causal):
    check(dev, 2, 300, 300, 3, 3, d, dtype, causal, buckets=32)


@pytest.mark.parametrize("buckets,md,causal", [(2, 2, True), (7, 20, True), (128, 256, True),
                                               (4, 3, False), (32, 16, False), (64, 256, False)])
def test_bias_shapes(dev, buckets, md, causal):
    check(dev, 2, 200, 333, 2, 1, 32, F32, causal, buckets=buckets, md=md)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("buckets", [0, 32])
def test_padded_batch(dev, dtype, buckets):
    check(dev, 5, 140, 140, 4, 2, 64, dtype, True, lengths=[140, 0, 1, 77, 128], buckets=buckets)
    check(dev, 3, 100, 210, 2, 2, 64, dtype, False, lengths=[100, 3, 64],
          k_lengths=[0, 210, 65], buckets=buckets)


def packed(dev, lens, k_lens, lead, tail, h, g, d, dtype, causal, buckets=0, layout="rows"):
    n, m = sum(lens) + lead + tail, sum(k_lens or lens) + lead + tail
    q, k, v, do = make((n,), (m,), h, g, d, dtype, dev, layout=layout)
    off = torch.tensor([0] + lens).cumsum(0) + lead
    koff = torch.tensor([0] + k_lens).cumsum(0) + lead if k_lens else off
    seqs = [(int(a), x, int(b), y) for a, x, b, y in zip(off, lens, koff, k_lens or lens)]
    bias = torch.randn(buckets, h, generator=torch.Generator().manual_seed(7)).to(dev) \
        .requires_grad_() if buckets else None
    ref = Ref(q, k, v, do, seqs, causal, d ** -0.5, bias)
    for x in (q, k, v):
        x.requires_grad_()
    out = slk.attention(q, k, v, causal=causal, offsets=off.int().to(dev),
                        k_offsets=koff.int().to(dev) if k_lens else None, bias=bias)
    leaves = [q, k, v] + ([bias] if buckets else [])
    grads = torch.autograd.grad(out, leaves, do)
    for name, x in zip(("out", "dq", "dk", "dv", "dbias"), (out, *grads)):
        close(name, x, ref, dtype)
    inside = torch.zeros(n, dtype=torch.bool)
    for q0, nq, _, _ in seqs:
        inside[q0:q0 + nq] = True
    assert (out.detach().cpu()[~inside] == 0).all() and (grads[0].cpu()[~inside] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_sequences(dev, dtype, causal):
    lens = [1, 130, 0, 64, 63, 65, 2, 200]
    packed(dev, lens, None, 0, 0, 4, 2, 64, dtype, causal)
    packed(dev, lens, None, 3, 17, 2, 1, 128, dtype, causal, buckets=32)
    packed(dev, lens, [5, 130, 9, 0, 200, 65, 1, 128], 0, 5, 2, 2, 64, dtype, causal,
           layout="cols")


def test_many_sequences(dev):
    """More sequences than the plan's workgroup has threads."""
    gen = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 6, (1500,), generator=gen).tolist()
    packed(dev, lens, None, 0, 1, 1, 1, 32, F32, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("b,t,s,h,g,d", [(3, 1, 100, 4, 1, 64), (2, 1, 3000, 8, 2, 128),
                                         (1, 1, 5001, 3, 3, 64), (2, 5, 700, 4, 2, 40),
                                         (1, 16, 2000, 2, 2, 128), (4, 2, 33, 6, 6, 32),
                                         (2, 3, 50, 2, 1, 33), (1, 1, 1, 1, 1, 1)])
@pytest.mark.parametrize("buckets", [0, 32])
def test_few_queries(dev, b, t, s, h, g, d, dtype, buckets):
    q, k, v, do = make((b, t), (b, s), h, g, d, dtype, dev)
    bias = torch.randn(buckets, h, device=dev) if buckets else None
    lens = [max(0, s - 37 * i) for i in range(b)]
    seqs = [(i * t, t, i * s, n) for i, n in enumerate(lens)]
    for causal in (True, False):
        ref = Ref(q, k, v, do, seqs, causal, d ** -0.5, bias)
        with torch.no_grad():
            out = slk.attention(q, k, v, causal=causal, bias=bias,
                                k_lengths=torch.tensor(lens, dtype=torch.int32, device=dev))
        close("out", out, ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_split_keys_of_a_prompt(dev, dtype):
    """Few query tiles over many keys: the keys are split over workgroups."""
    check(dev, 1, 70, 3001, 2, 1, 64, dtype, True)
    check(dev, 1, 70, 3001, 2, 1, 64, dtype, False, k_lengths=[1500])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_is_masked_may_hold_anything(dev, dtype, value):
    """Rows past a sequence's end, and keys (queries) that others do not see."""
    b, t, h, g, d = 2, 150, 2, 1, 64
    q, k, v, do = make((b, t), (b, t), h, g, d, dtype, dev)
    lens = [100, 150]
    ref = Ref(*(torch.nan_to_num(x) for x in (q, k, v, do)), [(0, 100, 0, 100), (t, 150, t, 150)],
              True, d ** -0.5)
    for x in (q, k, v, do):
        x[0, 100:] = value  # behind the first sequence's end
    for x in (q, k, v):
        x.requires_grad_()
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = slk.attention(q, k, v, lengths=n)
    grads = torch.autograd.grad(out, [q, k, v], do)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        close(name, x, ref, dtype)

    # a key (and its value) at position 90 reaches the queries from 90 on, no other
    at = 90
    k2, v2 = k.detach().clone(), v.detach().clone()
    k2[1, at], v2[1, at] = value, value
    k2.requires_grad_(), v2.requires_grad_(), q.requires_grad_()
    out2 = slk.attention(q, k2, v2, lengths=n)
    dq2, = torch.autograd.grad(out2, [q], do)
    for got, was in ((out2, out), (dq2, grads[0])):
        torch.testing.assert_close(got[0], was[0], rtol=0, atol=0)
        assert got[1, :at].isfinite().all()
        assert not got[1, at:].isfinite().any()
    torch.testing.assert_close(out2[1, :at], out[1, :at], rtol=2 ** -7, atol=1e-3)

    # a query (and its output's gradient) at position 90 reaches the keys up to 90
    q3, do3 = q.detach().clone(), do.clone()
    q3[1, at], do3[1, at] = value, value
    q3.requires_grad_()
    out3 = slk.attention(q3, k, v, lengths=n)
    dk3, dv3 = torch.autograd.grad(out3, [k, v], do3)
    assert out3[1, :at].isfinite().all() and out3[1, at + 1:].isfinite().all()
    for x in (dk3, dv3):
        assert x[1, at + 1:].isfinite().all() and not x[1, :at + 1].isfinite().any()
        assert x[0].isfinite().all()


@pytest.mark.parametrize("t", [1, 4])
def test_what_single_tokens_do_not_see_may_hold_anything(dev, t):
    q, k, v, do = make((2, t), (2, 300), 4, 2, 64, BF16, dev)
    n = torch.tensor([77, 300], dtype=torch.int32, device=dev)
    with torch.no_grad():
        clean = slk.attention(q, k, v, k_lengths=n)
        k[0, 77:], v[0, 77:] = float("nan"), float("inf")
        dirty = slk.attention(q, k, v, k_lengths=n)
    assert torch.equal(clean, dirty)


def test_gradients_against_differences(dev):
    """A step e of an input changes sum(out·do) by e·gradient + O(e^3) (a central
    difference); float32 results of about 10 are off by 1e-5, over 2e = 0.04: 1e-3 of noise
    and (e^2) of curvature against gradients of about 1."""
    q, k, v, do = make((1, 40), (1, 40), 2, 1, 64, F32, dev)
    bias = torch.randn(8, 2, device=dev)
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]

    def f(*x):
        return slk.attention(x[0], x[1], x[2], bias=x[3], max_distance=20)

    grads = torch.autograd.grad(f(*leaves), leaves, do)
    gen = torch.Generator().manual_seed(1)
    for i, x in enumerate(leaves):
        way = torch.randn(x.shape, generator=gen).to(dev)
        way /= way.norm()
        e = 0.02
        with torch.no_grad():
            hi = [y + e * way if j == i else y for j, y in enumerate(leaves)]
            lo = [y - e * way if j == i else y for j, y in enumerate(leaves)]
            diff = ((f(*hi).double() - f(*lo).double()) * do.double()).sum() / (2 * e)
        want = (grads[i].double() * way.double()).sum()
        assert abs(float(diff - want)) <= 5e-3 * (1 + float(grads[i].norm())), i


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_very_different_sizes(dev, dtype):
    """Values and output gradients over thirty powers of ten, sequence by sequence: each
    sequence is as exact as alone."""
    b, t, h, d = 6, 70, 2, 64
    q, k, v, do = make((b, t), (b, t), h, h, d, dtype, dev)
    for i in range(b):
        v[i] *= 10.0 ** (5 * (i - 3))
        do[i] *= 10.0 ** (4 * (3 - i))
    for x in (q, k, v):
        x.requires_grad_()
    out = slk.attention(q, k, v)
    grads = torch.autograd.grad(out, [q, k, v], do)
    for i in range(b):
        one = slice(i, i + 1)
        ref = Ref(q[one], k[one], v[one], do[one], [(0, t, 0, t)], True, d ** -0.5)
        for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            close(name, x[one], ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_scores(dev, dtype):
    """Scores of hundreds: one key takes all the weight."""
    q, k, v, do = make((1, 130), (1, 130), 2, 2, 64, dtype, dev)
    ref = Ref(q, k, v, do, [(0, 130, 0, 130)], True, 8.0)
    out = slk.attention(q, k, v, scale=8.0)
    close("out", out, ref, dtype)
    ref = Ref(q, k, v, do, [(0, 130, 0, 130)], True, 0.0)
    close("out", slk.attention(q, k, v, scale=0.0), ref, dtype)


def test_repeats_bit_for_bit(dev):
    q, k, v, do = make((700,), (700,), 4, 2, 64, F32, dev)
    bias = torch.randn(32, 4, device=dev)
    off = torch.tensor([0, 130, 131, 400, 690], dtype=torch.int32, device=dev)
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]

    def once():
        out = slk.attention(q, k, v, offsets=off, bias=bias)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    first = once()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_offsets_out_of_range_are_clamped(dev):
    q, k, v, _ = make((200,), (200,), 2, 2, 64, BF16, dev)

    def at(*o):
        return slk.attention(q, k, v, offsets=torch.tensor(o, dtype=torch.int32, device=dev))

    assert torch.equal(at(-5, 60, 40, 500), at(0, 60, 60, 200))
    b = [x.reshape(2, 100, 2, 64) for x in (q, k, v)]

    def n(*o):
        return slk.attention(*b, lengths=torch.tensor(o, dtype=torch.int32, device=dev))

    assert torch.equal(n(-3, 1000), n(0, 100))


def test_buckets():
    assert relative_buckets(16, 128) == (0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [torch.finfo(F32).min, -float("inf")])
def test_biases_that_hide(dev, dtype, value):
    """Buckets of the type's lowest value, and of minus infinity: what has another key to look
    at does not see them. Of the lowest value, a row that has nothing else sees all alike."""
    b, t, h, d = 1, 150, 2, 64
    q, k, v, do = make((b, t), (b, t), h, h, d, dtype, dev)
    bias = torch.randn(8, h, device=dev)
    bias[3:6] = value  # distances 3 to ..
    ref = Ref(q, k, v, do, [(0, t, 0, t)], True, d ** -0.5, bias.clamp(min=-1e30), 20)
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]
    out = slk.attention(q, k, v, bias=bias, max_distance=20)
    for n, x in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do))):
        got = x.detach().double().cpu().reshape(ref.val[n].shape)
        assert got.isfinite().all(), n
        off = (got - ref.val[n]).norm() / ref.val[n].norm()
        assert float(off) <= (1e-5 if dtype is F32 else 2.0 ** -7), n
    with torch.no_grad():
        all_low = torch.full_like(bias, value)
        out = slk.attention(q, k, v, bias=all_low, max_distance=20)
        if value > -float("inf"):
            mean = torch.cumsum(v.double(), 1) / torch.arange(1, t + 1, device=dev)[:, None, None]
            torch.testing.assert_close(out.double(), mean, rtol=2 ** -7, atol=2 ** -7)
        else:
            assert (out == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_without_gradients_feature_major(dev, dtype):
    lens = [70, 1, 0, 200, 33]
    n = sum(lens) + 9
    q, k, v, do = make((n,), (n,), 4, 2, 64, dtype, dev, layout="cols")
    off = torch.tensor([0] + lens).cumsum(0)
    ref = Ref(q, k, v, do, [(int(a), m, int(a), m) for a, m in zip(off, lens)], True, 0.125)
    with torch.no_grad():
        out = slk.attention(q, k, v, offsets=off.int().to(dev), feature_major=True)
    close("out", out, ref, dtype)
    assert out.stride(0) == 1 and out.flatten(1).t().is_contiguous()


def test_bias_gradient_of_many_pairs(dev):
    """The last bucket holds most pairs, and their dS cancel. dP, a sum of d products of
    normal values, is about sqrt(d) and off by 2^-23 of it or so; a row's weights sum to 1,
    and so is its sum of dS. At random that makes sqrt(rows) of them, four times for what is
    rare; an error of one sign would add up over all rows."""
    b, t, h, d = 16, 512, 4, 64
    q, k, v, do = make((b, t), (b, t), h, h, d, F32, dev)
    bias = torch.randn(32, h, device=dev)
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]
    out = slk.attention(q, k, v, bias=bias)
    got = torch.autograd.grad(out, leaves, do)[3]
    # every row's dS sum to 0, so all buckets of a head do
    most = 4 * 2.0 ** -23 * d ** 0.5 * (b * t) ** 0.5
    assert float(got.double().sum(0).abs().max()) <= most


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("start", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("d,gap", [(64, 8), (40, 4), (36, 0), (128, 1)])
def test_alignment(dev, d, gap, start, dtype):
    """Rows that begin at any element, heads a few elements apart: the same bits."""
    b, t, h = 2, 70, 2
    q, k, v, do = make((b, t), (b, t), h, h, d, dtype, dev)

    def shifted(x):
        buf = torch.full((b, t, h, d + gap), float("nan"), dtype=dtype, device=dev).flatten()
        buf = torch.cat([buf.new_full((start,), float("nan")), buf])
        y = buf[start:].view(b, t, h, d + gap)[..., :d]
        y.copy_(x)
        return y

    want = [x.clone().requires_grad_() for x in (q, k, v)]
    got = [shifted(x).requires_grad_() for x in (q, k, v)]
    a, c = slk.attention(*want), slk.attention(*got)
    assert torch.equal(a, c)
    for x, y in zip(torch.autograd.grad(a, want, do), torch.autograd.grad(c, got, shifted(do))):
        assert torch.equal(x, y)


@pytest.mark.parametrize("t", [2, 3])
def test_gradients_of_rows_with_few_keys(dev, t):
    """dP - rowsum(dO∘O) cancels where a row sees few keys: with O as it is rounded to
    bfloat16 these gradients were off by 0.004. A rounded result is off by anything up to
    2^-8 of itself, 2^-8 / sqrt(3) in the mean; weights and their gradients by 2^-12."""
    b, h, d = 400, 1, 64
    q, k, v, do = make((b, t), (b, t), h, h, d, BF16, dev)
    ref = Ref(q, k, v, do, [(i, t, i, t) for i in range(0, b * t, t)], True, d ** -0.5)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(slk.attention(*leaves), leaves, do)
    for n, x in zip(("dq", "dk", "dv"), got):
        want = ref.val[n]
        off = (x.double().cpu().reshape(want.shape) - want).norm() / want.norm()
        assert float(off) <= 2.0 ** -8 / 3 ** 0.5 + 2.0 ** -12, n


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[150], [3, 130, 1, 70]])
def test_gradients_where_all_biases_are_the_lowest_value(dev, dtype, lens):
    """Such a bias swallows every score: all keys that a query sees weigh the same, which is
    what queries of zeros make of them; dq and dv do not depend on the queries otherwise."""
    n, h, d = sum(lens), 2, 64
    q, k, v, do = make((n,), (n,), h, h, d, dtype, dev)
    off = torch.tensor([0] + lens).cumsum(0)
    seqs = [(int(a), m, int(a), m) for a, m in zip(off, lens)]
    ref = Ref(torch.zeros_like(q), k, v, do, seqs, True, d ** -0.5)
    bias = torch.full((8, h), torch.finfo(F32).min, device=dev)
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]
    out = slk.attention(q, k, v, offsets=off.int().to(dev), bias=bias, max_distance=20)
    dq, dk, dv, dbias = torch.autograd.grad(out, leaves, do)
    assert dk.isfinite().all() and dbias.isfinite().all()
    for name, x in (("out", out), ("dq", dq), ("dv", dv)):
        want = ref.val[name]
        off_by = (x.detach().double().cpu().reshape(want.shape) - want).norm() / want.norm()
        assert float(off_by) <= (1e-5 if dtype is F32 else 2.0 ** -8), name


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_sequences_than_the_plan_has_threads(dev, dtype):
    """1100 sequences, some empty, one with more tiles than the others together."""
    gen = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 4, (1100,), generator=gen).tolist()
    lens[517] = 700
    n = sum(lens) + 3
    q, k, v, do = make((n,), (n,), 2, 1, 32, dtype, dev)
    off = torch.tensor([0] + lens).cumsum(0)
    ref = Ref(q, k, v, do, [(int(a), m, int(a), m) for a, m in zip(off, lens)], True, 32 ** -0.5)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = slk.attention(q, k, v, offsets=off.int().to(dev))
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do))):
        close(name, x, ref, dtype)
