"""activation against its definition in float64, its 8-bit codes bit for bit, and
SparseLinear's kept inputs.

Bounds, u = 2^-24. The kept x is fixed to the last bit (one float32 operation after another),
so dx has only the slope's and the product's roundings: f and f' are a few operations on
exp or erfc, each good to a few u of its value, where the terms that are added reach |f| +
|x f'| + 1; exp's argument carries u of itself, |u2| <= 30 before the exponential has left
float32's range. 64u of those terms covers both; bfloat16 results are rounded once more, to 8
significant bits: half a step is finfo(bfloat16).eps / 2 = 2^-8 of the value.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import sparsecore_amd as slk
from sparsecore_amd.act import decode8, encode8

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# gelu through erfc: 1 + erf loses all digits of the left tail, in 64 bits too
KINDS = {"relu": F.relu, "silu": F.silu, "gelu": lambda x: 0.5 * x * torch.erfc(-x * 0.5 ** 0.5),
         "gelu_tanh": lambda x: F.gelu(x, approximate="tanh")}


def kept(x):
    """What 8 bits keep of x, in x's memory order, as the definition's float32 operations."""
    order = sorted(range(x.dim()), key=lambda i: -x.stride(i))
    flat = x.detach().permute(order).float().cpu()
    rows = F.pad(flat.reshape(-1), (0, -flat.numel() % 256)).view(-1, 256)
    top = torch.where(rows.isfinite(), rows.abs(), 0.0).amax(1, keepdim=True)
    ok = top >= 2.0 ** -100
    inv = torch.where(ok, torch.full_like(top, 127.0) / top, 0.0)
    step = torch.where(ok, top * torch.tensor(1.0 / 127.0), 0.0)
    y = torch.where(rows.isfinite(), torch.round(rows * inv) * step, float("nan"))
    y = y.view(-1)[:flat.numel()].view(flat.shape)
    back = sorted(range(x.dim()), key=lambda i: order[i])
    return y.permute(back)


def make(shape, dtype, dev, layout="rows", seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x, dy = (scale * torch.randn(*shape, generator=g)).to(dtype), torch.randn(*shape, generator=g).to(dtype)
    if layout == "cols":
        x, dy = (t.t().contiguous().t() for t in (x, dy))
    return x.to(dev), dy.to(dev)


def check(x, dy, kind, bits):
    dtype = x.dtype
    x = x.detach().requires_grad_()
    y = slk.activation(x, kind, save_bits=bits)
    dx, = torch.autograd.grad(y, [x], [dy])
    f = KINDS[kind]
    z = x.detach().double().cpu()
    k = (kept(x) if bits == 8 else x.detach().cpu()).double().requires_grad_()
    want_dx, = torch.autograd.grad(f(k), [k], dy.double().cpu())
    slope = want_dx / torch.where(dy.double().cpu() == 0, 1.0, dy.double().cpu())
    half = 0.0 if dtype is F32 else torch.finfo(dtype).eps / 2
    u = 64 * 2.0 ** -24
    for name, got, want, terms in (
            ("y", y, f(z), f(z).abs() + z.abs()),
            ("dx", dx, want_dx, dy.double().cpu().abs() * (1 + slope.abs() + k.detach().abs()))):
        off = (got.detach().double().cpu() - want).abs() - (u * terms + half * want.abs())
        assert float(off.max()) <= 0, (name, float(off.max()))
    assert y.stride() == x.stride() and dx.stride() == x.stride()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("shape,layout", [((1, 1), "rows"), ((3, 85), "cols"), ((16, 16), "rows"),
                                          ((7, 257), "rows"), ((33, 100), "cols"),
                                          ((5, 3, 70), "rows")])
def test_sizes(dev, shape, layout, kind, dtype, bits):
    check(*make(shape, dtype, dev, layout), kind, bits)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large(dev, dtype):
    """Past the size from which a wave takes four blocks, an odd number of elements."""
    x, dy = make((2049, 2051), dtype, dev)
    check(x, dy, "gelu", 8)


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_far_values(dev, kind):
    """Where exp, erfc and the cube leave float32."""
    x = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 12.0, -12.0, 90.0, -90.0, 1e4, -1e4, 3e15, -3e15,
                      1e38, -1e38], device=dev)
    for v in x:
        y = slk.activation(v.reshape(1).requires_grad_(), kind, save_bits=32)
        want = KINDS[kind](v.double().cpu())
        assert float((y.detach().double().cpu() - want).abs()) <= 1e-5 * float(want.abs()) + 1e-37
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(slk.activation(leaf, kind, save_bits=32).sum(), [leaf])
    z = x.double().cpu().requires_grad_()
    want, = torch.autograd.grad(KINDS[kind](z.clamp(-1e4, 1e4)).sum(), [z])
    want = torch.where(z.detach() > 1e4, 1.0, torch.where(z.detach() < -1e4, 0.0, want))
    torch.testing.assert_close(dx.double().cpu(), want, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_codes(dev, dtype):
    for shape in ((1,), (255,), (256,), (1000,), (300, 77)):
        x, _ = make(shape, dtype, dev, scale=3.0)
        x.view(-1)[::9] *= 1e-3
        codes, scales = encode8(x)
        got = decode8(codes, scales, x.shape)
        assert torch.equal(got.cpu(), kept(x))
        assert (got - x.float()).abs().max() <= x.float().abs().max() / 253


def test_codes_of_strange_blocks(dev):
    x = torch.randn(256 * 6, device=dev)
    x[0:256] = 0
    x[256:512] = 1e-38
    x[512:768] *= 2.0 ** 120
    x[800], x[900], x[1000] = float("nan"), float("inf"), -float("inf")
    x[1024:1280] = float("nan")
    x[1280:1536] = 1e-42
    got = decode8(*encode8(x), x.shape)
    assert torch.equal(got.isnan(), ~x.isfinite())
    assert torch.equal(torch.nan_to_num(got.cpu(), nan=7.0), torch.nan_to_num(kept(x), nan=7.0))
    assert (got[:512] == 0).all() and (got[1280:] == 0).all()
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(slk.activation(leaf, "gelu").sum(), [leaf])
    assert torch.equal(dx.isnan(), ~x.isfinite())


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_alignment_and_strides(dev, offset, dtype):
    base, dbase = make((1003 + offset,), dtype, dev)
    check(base[offset:], dbase[offset:], "silu", 8)
    x, dy = make((40, 30), dtype, dev)
    wide = torch.randn(40, 60, device=dev).to(dtype)[:, ::2]  # gaps: y is compact
    y = slk.activation(wide.requires_grad_(), "relu")
    assert y.is_contiguous() and torch.equal(y, torch.relu(wide))
    x = x.requires_grad_()  # a gradient in another layout than x
    a, = torch.autograd.grad(slk.activation(x, "gelu"), [x], [dy.t().contiguous().t()])
    b, = torch.autograd.grad(slk.activation(x, "gelu"), [x], [dy])
    assert torch.equal(a, b)


def test_empty(dev):
    x = torch.empty(0, 8, device=dev, requires_grad=True)
    y = slk.activation(x)
    assert y.shape == x.shape
    assert torch.autograd.grad(y.sum(), [x])[0].shape == x.shape


def test_what_is_kept(dev):
    """A byte an element and a scale a block; x itself is free behind the call."""
    x = torch.randn(1 << 22, device=dev)
    leaf = x.requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = slk.activation(leaf * 1.0, "gelu")
    kept_bytes = torch.cuda.memory_allocated() - before - y.numel() * 4
    assert kept_bytes <= y.numel() * (1 + 4 / 256) + 4096


@pytest.mark.parametrize("shape", [(300, 96, 64), (40, 64, 10), (2000, 512, 256)])
def test_sparse_linear_keeps_its_input_in_8_bits(dev, shape):
    """Output and input gradient bit for bit as without, the weights' gradient that of the
    kept input, bit for bit."""
    n, k, m = shape
    torch.manual_seed(0)
    layer = slk.SparseLinear(k, m, sparsity=0.8).to(dev)
    x = torch.randn(n, k, device=dev, requires_grad=True)
    up = torch.randn(n, m, device=dev)

    def once(inp):
        y = layer(inp)
        return [y.detach(), *torch.autograd.grad(y, [layer._values, layer.bias, inp], up)]

    y, dw, db, dx = once(x)
    layer.save_bits = 8
    y8, dw8, db8, dx8 = once(x)
    assert torch.equal(y, y8) and torch.equal(dx, dx8) and torch.equal(db, db8)
    assert not torch.equal(dw, dw8)
    cols = x.detach().t().contiguous()
    seen = decode8(*encode8(cols), cols.shape).t().requires_grad_()
    layer.save_bits = 32
    assert torch.equal(once(seen)[1], dw8)


def test_sparse_linear_arguments(dev):
    with pytest.raises(ValueError, match="save_bits"):
        slk.SparseLinear(8, 8, save_bits=4)
    layer = slk.SparseLinear(8, 8, save_bits=8).to(dev)
    assert "save_bits=8" in layer.extra_repr()
    with torch.no_grad():
        layer(torch.randn(3, 8, device=dev))
    layer._values.requires_grad_(False)
    x = torch.randn(3, 8, device=dev, requires_grad=True)
    layer(x).sum().backward()
    assert x.grad is not None
