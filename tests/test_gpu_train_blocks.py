"""attention, its position bias and 8-bit activations as a training step uses them together:
the example's model against the same model in plain torch, captured steps, streams, and the
calls around autograd."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

import sparsecore_amd as slk
from sparsecore_amd.attn import relative_buckets

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parent.parent / "examples" / "train_char_gpt.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_char_gpt_blocks", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_forward(model, idx, target):
    x = model.tok(idx) + model.pos(torch.arange(idx.shape[1], device=idx.device))
    t = idx.shape[1]
    away = torch.arange(t, device=x.device)[:, None] - torch.arange(t, device=x.device)
    for blk in model.blocks:
        d = x.shape[-1]
        y = F.layer_norm(x, (d,), blk.norm1.weight, blk.norm1.bias)
        b = x.shape[0]
        q, k, v = (z.reshape(b, t, blk.heads, d // blk.heads).transpose(1, 2)
                   for z in blk.qkv(y).chunk(3, dim=-1))
        s = q @ k.transpose(2, 3) * (d // blk.heads) ** -0.5
        if model.rel is not None:
            starts = torch.tensor(relative_buckets(model.rel.shape[0], 64), device=x.device)
            which = torch.searchsorted(starts, away.clamp(0, 64), right=True) - 1
            s = s + model.rel.t()[:, which]
        a = torch.softmax(s.masked_fill(away < 0, -float("inf")), -1) @ v
        x = x + blk.out(a.transpose(1, 2).reshape(b, t, d))
        y = F.layer_norm(x, (d,), blk.norm2.weight, blk.norm2.bias)
        x = x + blk.down(F.gelu(blk.up(y)))
    y = F.layer_norm(x, (d,), model.norm.weight, model.norm.bias)
    return F.cross_entropy((y @ model.head.t()).reshape(-1, model.head.shape[0]),
                           target.reshape(-1))


@pytest.mark.parametrize("buckets", [0, 16])
def test_model_matches_plain_torch(dev, example, buckets):
    """Loss and every gradient, float32 both ways: two orders of the same sums through two
    blocks, within 1e-4 of each gradient's root mean square."""
    torch.manual_seed(0)
    model = example.CharGPT(70, 64, buckets=buckets).to(dev)
    if buckets:
        with torch.no_grad():
            model.rel.normal_()
    g = torch.Generator().manual_seed(1)
    idx, target = (torch.randint(0, 70, (8, 64), generator=g).to(dev) for _ in range(2))
    ours, theirs = model(idx, target), plain_forward(model, idx, target)
    torch.testing.assert_close(ours, theirs, rtol=1e-5, atol=0)
    params = list(model.parameters())
    a, b = torch.autograd.grad(ours, params), torch.autograd.grad(theirs, params)
    for (name, p), x, y in zip(model.named_parameters(), a, b):
        off = (x - y).abs().max()
        assert float(off) <= 1e-4 * float(y.square().mean().sqrt()) + 1e-9, name


def test_blocks_in_8_bits(dev, example):
    """With act_bits=8 the loss is the same to the last bit (forwards read x itself) and every
    gradient is near the other's: a kept value is off by at most 1/254 of its block's largest,
    uniformly, 1/440 of it in the root mean square; blocks of 256 normal values reach about 3
    deviations, so 0.7% of a value's deviation for each of the five kept tensors of a block,
    two blocks: 2.2% if independent, 5% allowed."""
    g = torch.Generator().manual_seed(1)
    idx, target = (torch.randint(0, 70, (8, 64), generator=g).to(dev) for _ in range(2))
    out = []
    for bits in (32, 8):
        torch.manual_seed(0)
        model = example.CharGPT(70, 64, act_bits=bits, buckets=16).to(dev)
        loss = model(idx, target)
        out.append((loss.detach(), torch.autograd.grad(loss, list(model.parameters()))))
    assert torch.equal(out[0][0], out[1][0])
    for (name, _), x, y in zip(model.named_parameters(), out[0][1], out[1][1]):
        assert float((x - y).norm()) <= 0.05 * float(x.norm()) + 1e-12, name


def test_training_runs_and_repeats(dev, example):
    a = example.train(steps=15, state_bits=8, act_bits=8, buckets=16)
    assert a == example.train(steps=15, state_bits=8, act_bits=8, buckets=16)
    assert all(x == x for x in a)


def inputs(dev, n=200, h=4, g=2, d=64, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(n, h, d, generator=gen).to(dtype).to(dev) for _ in range(2))
    k, v = (torch.randn(n, g, d, generator=gen).to(dtype).to(dev) for _ in range(2))
    bias = torch.randn(16, h, generator=gen).to(dev)
    off = torch.tensor([0, 70, 71, 190], dtype=torch.int32, device=dev)
    return q, k, v, do, bias, off


def step(q, k, v, do, bias, off):
    out = slk.attention(q, k, v, offsets=off, bias=bias)
    y = slk.activation(out, "gelu")
    return [y, *torch.autograd.grad(y, [q, k, v, bias], do)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(dev, dtype):
    """Forward and backward in a graph, replayed with new values, lengths included, and eager
    work between the replays."""
    q, k, v, do, bias, off = inputs(dev, dtype=dtype)
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(q, k, v, do, bias, off)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, k, v, do, bias, off)
    for i in range(4):
        new = inputs(dev, dtype=dtype, seed=i + 1)
        with torch.no_grad():
            for x, y in zip((q, k, v, do, bias), new):
                x.copy_(y)
            off.copy_(torch.tensor([0, 3 * i, 100 + i, 200], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        seen = [x.clone() for x in got]
        fresh = [x.detach().clone().requires_grad_() for x in leaves]
        want = step(*fresh[:3], do.clone(), fresh[3], off.clone())
        assert all(torch.equal(a, b) for a, b in zip(seen, want)), i


def test_captured_steps_hold_kernels_only(dev):
    from sparsecore_amd import _lib

    q, k, v, do, bias, off = inputs(dev)
    for x in (q, k, v, bias):
        x.requires_grad_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        step(q, k, v, do, bias, off)
    assert set(_lib.graph_node_types(graph)) <= {"kernel", "empty"}


def test_two_captured_graphs_share_nothing(dev):
    """Two graphs captured one after the other, replayed in turn: each its own results."""
    a, b = inputs(dev, seed=1), inputs(dev, seed=2)
    graphs = []
    for x in (a, b):
        for t in (*x[:3], x[4]):
            t.requires_grad_()
        want = [t.detach().clone() for t in step(*x)]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step(*x)
        graphs.append((g, got, want))
    for _ in range(3):
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, got, want in graphs:
            assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_streams(dev):
    """Calls in flight on several streams at once, each with its own values."""
    sets = [inputs(dev, seed=i) for i in range(3)]
    for x in sets:
        for t in (*x[:3], x[4]):
            t.requires_grad_()
    want = [step(*x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, x in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append([step(*x) for _ in range(4)])
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_gradients_of_some_inputs(dev):
    q, k, v, do, bias, off = inputs(dev)
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]
    out = slk.attention(q, k, v, offsets=off, bias=bias)
    want = torch.autograd.grad(out, leaves, do)
    for wanted in ([0], [1], [2], [3], [0, 3], [1, 2], [2, 3]):
        xs = [x.detach().clone().requires_grad_(i in wanted) for i, x in enumerate(leaves)]
        out = slk.attention(*xs[:3], offsets=off, bias=xs[3])
        for i, g in zip(wanted, torch.autograd.grad(out, [xs[i] for i in wanted], do)):
            assert torch.equal(g, want[i]), (wanted, i)


def test_the_same_graph_twice(dev):
    q, k, v, do, bias, off = inputs(dev)
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]
    out = slk.attention(q, k, v, offsets=off, bias=bias)
    a = torch.autograd.grad(out, leaves, do, retain_graph=True)
    other = torch.autograd.grad(out, leaves, torch.full_like(do, float("nan")), retain_graph=True)
    b = torch.autograd.grad(out, leaves, do)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert other[0][:190].isnan().all()
    x = torch.randn(300, device=dev, requires_grad=True)
    y = slk.activation(x)
    a, = torch.autograd.grad(y.sum(), [x], retain_graph=True)
    b, = torch.autograd.grad(y.sum(), [x])
    assert torch.equal(a, b)


def test_one_tensor_in_several_places(dev):
    x = torch.randn(2, 50, 2, 64, device=dev, requires_grad=True)
    do = torch.randn_like(x)
    got, = torch.autograd.grad(slk.attention(x, x, x), [x], do)
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    want = sum(torch.autograd.grad(slk.attention(*parts), parts, do))
    torch.testing.assert_close(got, want, rtol=1e-6, atol=1e-6)


def test_broadcast_inputs_and_gradients(dev):
    """Keys shared by all entries (stride 0), and the gradient of a sum (all strides 0)."""
    q = torch.randn(3, 40, 2, 64, device=dev, requires_grad=True)
    k, v = (torch.randn(1, 90, 1, 64, device=dev, requires_grad=True) for _ in range(2))
    out = slk.attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), causal=False)
    got = torch.autograd.grad(out.sum(), [q, k, v])
    kk, vv = (x.detach().repeat(3, 1, 1, 1).requires_grad_() for x in (k, v))
    out2 = slk.attention(q, kk, vv, causal=False)
    assert torch.equal(out, out2)
    want = torch.autograd.grad(out2, [q, kk, vv], torch.ones_like(out2))
    assert torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):
        torch.testing.assert_close(a, b.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)


def test_second_derivatives_are_refused(dev):
    q, k, v = (torch.randn(1, 8, 1, 32, device=dev, requires_grad=True) for _ in range(3))
    g, = torch.autograd.grad(slk.attention(q, k, v).sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [q])


def test_an_output_changed_in_place_is_noticed(dev):
    q, k, v = (torch.randn(1, 8, 1, 32, device=dev, requires_grad=True) for _ in range(3))
    out = slk.attention(q, k, v)
    with torch.no_grad():
        out.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        out.sum().backward()


def test_inputs_may_change_behind_the_forward(dev):
    """q, k and v are kept packed: what happens to them later is no matter."""
    q, k, v, do, bias, off = inputs(dev)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(slk.attention(q, k, v, offsets=off), leaves, do)
    out = slk.attention(q, k, v, offsets=off)
    with torch.no_grad():
        for x in leaves:
            x.fill_(float("nan"))
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, leaves, do)))


@pytest.mark.parametrize("shape", [(0, 5, 2, 32), (2, 0, 2, 32)])
def test_no_queries(dev, shape):
    q = torch.randn(*shape, device=dev, requires_grad=True)
    k, v = (torch.randn(shape[0], 7, 1, 32, device=dev, requires_grad=True) for _ in range(2))
    bias = torch.randn(8, 2, device=dev, requires_grad=True)
    out = slk.attention(q, k, v, bias=bias, max_distance=20)
    assert out.shape == q.shape
    dq, dk, dv, db = torch.autograd.grad(out.sum(), [q, k, v, bias])
    assert dq.shape == q.shape and (dk == 0).all() and (dv == 0).all() and (db == 0).all()


def test_no_keys(dev):
    q = torch.randn(2, 5, 2, 32, device=dev, requires_grad=True)
    k, v = (torch.randn(2, 0, 1, 32, device=dev, requires_grad=True) for _ in range(2))
    bias = torch.randn(8, 2, device=dev, requires_grad=True)
    out = slk.attention(q, k, v, causal=False, bias=bias, max_distance=20)
    assert (out == 0).all()
    dq, dk, dv, db = torch.autograd.grad(out.sum(), [q, k, v, bias])
    assert (dq == 0).all() and dk.shape == k.shape and (db == 0).all()
    with torch.no_grad():
        assert (slk.attention(q, k, v) == 0).all()
    none = torch.zeros(1, dtype=torch.int32, device=dev)
    x = torch.randn(9, 2, 32, device=dev)
    assert (slk.attention(x, x, x, offsets=none) == 0).all()


def test_far_apart_in_memory(dev):
    """Rows whose places differ by more than 2^32 elements: keys of single tokens, packed
    operands, outputs and gradients."""
    step_ = 40_000_000
    room = torch.empty(120 * step_ + 64, dtype=torch.bfloat16, device=dev)  # 9.6 GB
    far = room.as_strided((1, 120, 1, 64), (0, step_, 64, 1))
    near = torch.randn(1, 120, 1, 64, device=dev).to(torch.bfloat16)
    far.copy_(near)
    q = torch.randn(1, 120, 1, 64, device=dev).to(torch.bfloat16)
    with torch.no_grad():
        for x in (q, q[:, :1]):
            assert torch.equal(slk.attention(x, far, far), slk.attention(x, near, near))
        assert torch.equal(slk.attention(far, near, near), slk.attention(near, near, near))


@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16])
def test_bias_types_and_strides(dev, bias_dtype):
    q, k, v, do, bias, off = inputs(dev, dtype=torch.bfloat16)
    bias = bias.to(bias_dtype)
    across = bias.t().contiguous().t().requires_grad_()
    flat = bias.clone().requires_grad_()
    got = slk.attention(q, k, v, offsets=off, bias=across)
    want = slk.attention(q, k, v, offsets=off, bias=flat)
    assert torch.equal(got, want)
    a, = torch.autograd.grad(got, [across], do)
    b, = torch.autograd.grad(want, [flat], do)
    assert a.dtype == bias_dtype and torch.equal(a, b)


def test_refusals(dev):
    q = torch.randn(2, 10, 4, 64, device=dev)
    k = torch.randn(2, 10, 2, 64, device=dev)
    n = torch.tensor([3, 4], dtype=torch.int32, device=dev)

    def no(match, *a, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            slk.attention(*a, **kw)

    no("Tensor", q, k, 3, error=TypeError)
    no("HIP", q, k, k.cpu(), error=RuntimeError)
    no("float32 or all bfloat16", q, k, k.bfloat16())
    no("float32 or all bfloat16", q.double(), k.double(), k.double())
    no("must be", q[0], k, k)
    no("must be", q, k, k[:, :5])
    no("entries", q[:1], k, k)
    no("head size", q, k[..., :32], k[..., :32])
    no("head size", *(torch.randn(1, 4, 1, 136, device=dev),) * 3)
    no("multiple", q[:, :, :3], k, k)
    no("not both", q[0], k[0], k[0], offsets=n, lengths=n)
    no("share offsets", q[0], k[0, :5], k[0, :5], offsets=n)
    no("need offsets", q, k, k, k_offsets=n)
    no("int32", q, k, k, lengths=n.long())
    no("int32", q, k, k, lengths=n[:1])
    no("same length", q[0], k[0], k[0], offsets=n, k_offsets=n[:1])
    no("buckets", q, k, k, bias=torch.zeros(1, 4, device=dev))
    no("buckets", q, k, k, bias=torch.zeros(130, 4, device=dev))
    no("buckets", q, k, k, bias=torch.zeros(5, 4, device=dev), causal=False)
    no("buckets, 4", q, k, k, bias=torch.zeros(8, 3, device=dev))
    no("float32 or", q.bfloat16(), k.bfloat16(), k.bfloat16(), bias=torch.zeros(8, 4, device=dev).half())
    no("max_distance", q, k, k, bias=torch.zeros(8, 4, device=dev), max_distance=300)
    no("above 16", q, k, k, bias=torch.zeros(32, 4, device=dev), max_distance=16)
    no("scale", q, k, k, scale=-1.0)
    no("scale", q, k, k, scale=float("nan"))
    x = torch.randn(4, device=dev)
    for bad, kw in ((x.cpu(), {}), (x.double(), {}), (x, {"kind": "tanh"}), (x, {"save_bits": 4}),
                    (x, {"kind": "none"})):
        with pytest.raises((RuntimeError, ValueError)):
            slk.activation(bad, **kw)
    with pytest.raises(TypeError):
        slk.activation([1.0])
