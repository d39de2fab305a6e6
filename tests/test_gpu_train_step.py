"""The training step that the operators make together: the example's model against the
same model written with torch's own norm, loss and residual sums, and its training."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

import sparsecore_amd as slk

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parent.parent / "examples" / "train_char_gpt.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_char_gpt", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_forward(model, idx, target):
    x = model.tok(idx) + model.pos(torch.arange(idx.shape[1], device=idx.device))
    for blk in model.blocks:
        d = x.shape[-1]
        y = F.layer_norm(x, (d,), blk.norm1.weight, blk.norm1.bias)
        b, t, _ = x.shape
        q, k, v = (z.reshape(b, t, blk.heads, d // blk.heads).transpose(1, 2)
                   for z in blk.qkv(y).chunk(3, dim=-1))
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        x = x + blk.out(a.transpose(1, 2).reshape(b, t, d))
        y = F.layer_norm(x, (d,), blk.norm2.weight, blk.norm2.bias)
        x = x + blk.down(F.gelu(blk.up(y)))
    y = F.layer_norm(x, (d,), model.norm.weight, model.norm.bias)
    return F.cross_entropy((y @ model.head.t()).reshape(-1, model.head.shape[0]),
                           target.reshape(-1))


def test_model_matches_plain_torch(dev, example):
    """Loss and every gradient, float32 both ways: two orders of the same sums through two
    blocks, within 1e-4 of each gradient's root mean square."""
    torch.manual_seed(0)
    model = example.CharGPT(70, 64).to(dev)
    g = torch.Generator().manual_seed(1)
    idx, target = (torch.randint(0, 70, (8, 64), generator=g).to(dev) for _ in range(2))
    ours, theirs = model(idx, target), plain_forward(model, idx, target)
    torch.testing.assert_close(ours, theirs, rtol=1e-5, atol=0)
    params = list(model.parameters())
    a, b = torch.autograd.grad(ours, params), torch.autograd.grad(theirs, params)
    for (name, p), x, y in zip(model.named_parameters(), a, b):
        off = (x - y).abs().max()
        assert float(off) <= 1e-4 * float(y.square().mean().sqrt()) + 1e-9, name


@pytest.mark.parametrize("bits", [32, 8])
def test_training_learns_through_rewrites(dev, example, bits):
    losses = example.train(steps=120, state_bits=bits)
    first, last = sum(losses[:5]) / 5, sum(losses[-5:]) / 5
    assert all(x == x for x in losses)
    assert last < 0.75 * first, (first, last)


def test_training_repeats(dev, example):
    assert example.train(steps=20) == example.train(steps=20)


def test_residual_norm_module(dev):
    torch.manual_seed(0)
    m = slk.ResidualNorm(96, "rms", post=True, gate=0.5, scale=2.0).to(dev)
    x, u = torch.randn(5, 96, device=dev), torch.randn(5, 96, device=dev)
    r, y = m(x, u)
    want = x + 2.0 * 0.5 * F.rms_norm(u, (96,), eps=1e-5)
    torch.testing.assert_close(r, want, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(y, F.rms_norm(want, (96,), eps=1e-5), rtol=1e-5, atol=1e-5)
    assert sorted(k for k, _ in m.named_parameters()) == ["gate", "post_weight", "weight"]
    r, y = m(x)
    assert r is x
    with pytest.raises(ValueError, match="kind"):
        slk.ResidualNorm(96, "group")
