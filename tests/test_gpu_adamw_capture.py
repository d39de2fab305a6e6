"""A captured AdamW step beside topology rewrites, checkpoints and copies."""

from __future__ import annotations

import pytest
import torch

import sparsecore_amd as slk

pytestmark = pytest.mark.gpu


def capture(step):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    return graph


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_after_rewrites_are_eager_steps(dev, bits):
    """Gradients are written into the tensors that the capture read; each rewrite is
    followed by follow() on one side and found by the eager step on the other."""
    nets, opts, algos = [], [], []
    for k in range(2):
        torch.manual_seed(0)
        net = slk.SparseLinear(96, 80, sparsity=0.8, bias=False).to(dev)
        net._values.grad = torch.zeros_like(net._values)
        opt = slk.AdamW(net.parameters(), lr=1e-2, state_bits=bits, capturable=True)
        net.apply(opt.attach)
        algo = slk.SET(sparsity=0.8, drop_fraction=0.3, update_freq=2, seed=1)
        net.apply(algo)
        nets.append(net), opts.append(opt), algos.append(algo)
    graph, gen = None, torch.Generator().manual_seed(2)
    for step in range(7):
        g = torch.randn(nets[0]._values.numel(), generator=gen).to(dev)
        for net in nets:  # padding slots have gradient 0
            live = net._csr.col_indices >= 0
            net._values.grad.copy_(torch.where(live, g.view_as(net._values), 0.0))
        opts[0].step()
        if step == 0:
            opts[1].step()
        else:
            opts[1].follow()
            if graph is None:
                graph = capture(opts[1].step)
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(nets[0]._values, nets[1]._values), step
        for k, v in opts[0].state[nets[0]._values].items():
            assert torch.equal(v, opts[1].state[nets[1]._values][k]), (step, k)
        old = nets[0]._csr.col_indices.clone()
        for algo in algos:
            algo.step()
        assert torch.equal(nets[0]._csr.col_indices, nets[1]._csr.col_indices)
        if step % 2:
            assert not torch.equal(old, nets[0]._csr.col_indices)


def test_captures_that_would_repeat_a_beginning_or_a_move_are_refused(dev):
    net = slk.SparseLinear(96, 80, sparsity=0.8, bias=False).to(dev)
    net._values.grad = torch.zeros_like(net._values)
    opt = slk.AdamW(net.parameters(), capturable=True)
    net.apply(opt.attach)
    with pytest.raises(RuntimeError, match="before capturing"):
        capture(opt.step)
    opt.step()
    algo = slk.SET(sparsity=0.8, drop_fraction=0.3, update_freq=1, seed=1)
    net.apply(algo)
    algo.step()
    with pytest.raises(RuntimeError, match="follow"):
        capture(opt.step)
    opt.follow()
    capture(opt.step).replay()
    torch.cuda.synchronize()
    assert float(opt.state[net._values]["step"]) == 2


def test_a_backward_across_a_step_is_refused(dev):
    """SparseLinear's backward and that of linear_cross_entropy over few tokens read the
    weights themselves."""
    net = slk.SparseLinear(64, 48, sparsity=0.5, bias=False).to(dev)
    head = torch.nn.Parameter(torch.randn(100, 64, device=dev))
    x = torch.randn(8, 64, device=dev, requires_grad=True)
    t = torch.zeros(8, dtype=torch.int64, device=dev)
    for p, loss in ((net._values, lambda: net(x).square().sum()),
                    (head, lambda: slk.linear_cross_entropy(x, head, t))):
        opt = slk.AdamW([p])
        late = loss()
        loss().backward()
        opt.step()
        with pytest.raises(RuntimeError, match="inplace"):
            late.backward()
        opt.zero_grad()
