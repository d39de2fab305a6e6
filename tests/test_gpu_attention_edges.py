"""attention at its edges: calls without queries or without keys, and some of the gradients."""

from __future__ import annotations

import pytest
import torch

import sparsecore_amd as slk

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def leave_garbage(dev, nbytes=1 << 20):
    """Freed blocks of several sizes that hold ones in every bit: what the next call's saved
    and scratch memory may hold."""
    sizes = [nbytes >> i for i in range(12)]
    blocks = [torch.full((n,), 0xff, dtype=torch.uint8, device=dev) for n in sizes for _ in "123"]
    torch.cuda.synchronize()
    del blocks


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("buckets", [0, 8])
@pytest.mark.parametrize("h,g,s", [(2, 2, 7), (4, 1, 300), (6, 2, 129)])
@pytest.mark.parametrize("mode", ["whole", "lengths", "k_lengths", "packed"])
def test_no_queries_in_any_layout(dev, mode, h, g, s, buckets, causal, dtype):
    leave_garbage(dev)
    d, b = 32, 3
    lead_q, lead_k = ((0,), (3 * s,)) if mode == "packed" else ((b, 0), (b, s))
    q = torch.randn(*lead_q, h, d, device=dev).to(dtype).requires_grad_()
    k, v = (torch.randn(*lead_k, g, d, device=dev).to(dtype).requires_grad_() for _ in range(2))
    bias = torch.randn(buckets, h, device=dev, requires_grad=True) if buckets else None
    ints = torch.tensor([s, 0, s // 2], dtype=torch.int32, device=dev)
    more = {"whole": {}, "lengths": {"lengths": torch.zeros_like(ints), "k_lengths": ints},
            "k_lengths": {"k_lengths": ints},
            "packed": {"offsets": torch.zeros(4, dtype=torch.int32, device=dev),
                       "k_offsets": torch.tensor([2, s, s, 2 * s], dtype=torch.int32,
                                                 device=dev)}}[mode]
    out = slk.attention(q, k, v, causal=causal, bias=bias, max_distance=20, **more)
    assert out.shape == q.shape
    leaves = [q, k, v] + ([bias] if buckets else [])
    grads = torch.autograd.grad(out, leaves, torch.empty_like(out))
    for x, y in zip(grads, leaves):
        assert x.shape == y.shape and x.dtype == y.dtype and (x == 0).all()


@pytest.mark.parametrize("buckets", [0, 8])
def test_packed_batch_of_nothing(dev, buckets):
    """No sequences, and sequences that are all empty, with rows of none behind them."""
    for off in ([0], [0, 0, 0], [4, 4]):
        for rows in (0, 9):
            leave_garbage(dev)
            x = torch.randn(rows, 2, 32, device=dev, requires_grad=True)
            bias = torch.randn(buckets, 2, device=dev, requires_grad=True) if buckets else None
            out = slk.attention(x, x, x, bias=bias, max_distance=20,
                                offsets=torch.tensor(off, dtype=torch.int32, device=dev))
            leaves = [x] + ([bias] if buckets else [])
            assert (out == 0).all()
            for g, y in zip(torch.autograd.grad(out, leaves, torch.ones_like(out)), leaves):
                assert g.shape == y.shape and (g == 0).all()


def test_no_queries_captured(dev):
    """The same in a graph, replayed with other lengths."""
    k, v = (torch.randn(2, 70, 2, 64, device=dev, requires_grad=True) for _ in range(2))
    q = torch.randn(2, 0, 2, 64, device=dev)
    n = torch.tensor([70, 3], dtype=torch.int32, device=dev)

    def step():
        out = slk.attention(q, k, v, k_lengths=n)
        return torch.autograd.grad(out, [k, v], torch.empty_like(out))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        for x in got:
            x.fill_(1.0)
        n.copy_(torch.tensor([20 * i, 70 - i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all((x == 0).all() for x in got)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mode", ["whole", "k_lengths", "packed"])
@pytest.mark.parametrize("buckets", [0, 8])
def test_no_keys_in_any_layout(dev, mode, buckets, dtype):
    leave_garbage(dev)
    b, t, h, d = 3, 70, 2, 32
    lead_q, lead_k = ((b * t,), (0,)) if mode == "packed" else ((b, t), (b, 0))
    q = torch.randn(*lead_q, h, d, device=dev).to(dtype).requires_grad_()
    k, v = (torch.randn(*lead_k, 1, d, device=dev).to(dtype).requires_grad_() for _ in range(2))
    bias = torch.randn(buckets, h, device=dev, requires_grad=True) if buckets else None
    zeros = torch.zeros(4, dtype=torch.int32, device=dev)
    more = {"whole": {}, "k_lengths": {"k_lengths": zeros[:3]},
            "packed": {"offsets": torch.tensor([3, t, t, 2 * t], dtype=torch.int32, device=dev),
                       "k_offsets": zeros}}[mode]
    out = slk.attention(q, k, v, bias=bias, max_distance=20, **more)
    assert (out == 0).all()
    leaves = [q, k, v] + ([bias] if buckets else [])
    for x, y in zip(torch.autograd.grad(out, leaves, torch.ones_like(out)), leaves):
        assert x.shape == y.shape and (x == 0).all()


@pytest.mark.parametrize("uneven", [False, True])
@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (1, 2), (0, 3)])
def test_some_of_the_gradients(dev, wanted, uneven):
    """Any of them alone has the bits that it has among all."""
    t, h, d = 200, 4, 64
    gen = torch.Generator().manual_seed(0)
    q, k, v, bias = (torch.randn(*s, generator=gen) for s in ((1, t, h, d), (1, t, 2, d),
                                                              (1, t, 2, d), (8, h)))
    if uneven:
        q[:, ::7] *= 2.0 ** -20
        v[:, ::5] *= 2.0 ** 20
    do = torch.randn(1, t, h, d, generator=gen).to(dev)
    leaves = [x.to(dev) for x in (q, k, v, bias)]

    def grads(of):
        x = [y.clone().requires_grad_(i in of) for i, y in enumerate(leaves)]
        out = slk.attention(*x[:3], bias=x[3], max_distance=20)
        return torch.autograd.grad(out, [x[i] for i in of], do)

    among_all = grads((0, 1, 2, 3))
    for i, x in zip(wanted, grads(wanted)):
        assert torch.equal(x, among_all[i]), i


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("mode,t,s", [("batch", 1, 1), ("batch", 70, 1), ("batch", 150, 150),
                                      ("batch", 100, 40), ("packed", 35, 35), ("lengths", 9, 9)])
@pytest.mark.parametrize("uneven", [False, True])
def test_rows_that_see_a_single_key(dev, mode, t, s, causal, uneven, dtype):
    """Their weight is 1 whatever the scores are: no gradient goes to the query, none through
    it to the key or to the bias. Exactly none."""
    gen = torch.Generator().manual_seed(0)
    h, d, b = 2, 64, 1 if mode == "packed" else 3
    lead_q, lead_k = ((t,), (s,)) if mode == "packed" else ((b, t), (b, s))
    q, do = (torch.randn(*lead_q, h, d, generator=gen).to(dtype).to(dev) for _ in range(2))
    k, v = (torch.randn(*lead_k, 1, d, generator=gen).to(dtype).to(dev) for _ in range(2))
    if uneven:
        v[..., 0, 0, :] *= 2.0 ** 30
        do[..., -1, :, :] *= 2.0 ** -30
    bias = torch.randn(8, h, generator=gen).to(dev)
    more = {"packed": {"offsets": torch.arange(t + 1, dtype=torch.int32, device=dev)},
            "lengths": {"k_lengths": torch.ones(b, dtype=torch.int32, device=dev),
                        "lengths": torch.full((b,), t, dtype=torch.int32, device=dev)},
            "batch": {}}[mode]
    leaves = [x.requires_grad_() for x in (q, k, v, bias)]
    out = slk.attention(q, k, v, bias=bias, causal=causal, max_distance=20, **more)
    dq, dk, dv, dbias = torch.autograd.grad(out, leaves, do)
    if mode == "packed" or mode == "lengths" or s == 1:
        assert (dq == 0).all() and (dk == 0).all() and (dbias == 0).all()
    elif causal:
        first = max(0, t - s)  # the first query that sees a key
        assert (dq[:, :first + 1] == 0).all() and not (dq[:, first + 1:] == 0).all()
        # what that query leaves the first key: nothing but by its value
        do2 = do.clone()
        do2[:, first] *= 3.0
        other = torch.autograd.grad(slk.attention(q, k, v, bias=bias, max_distance=20, **more),
                                    leaves, do2)
        assert torch.equal(dq, other[0]) and not torch.equal(dv, other[2])
        torch.testing.assert_close(dk[:, 0], other[1][:, 0], rtol=2 ** -7, atol=1e-6)
    assert not (dv == 0).all()
