"""activation in bfloat16 where f is small: each result against its own size.

Bounds. A result is rounded to bfloat16, half a step: 2^-8 of it. Before that, the
exponential's argument, up to 113 in units of log 2 here, is rounded three times, 2.5 · 2^-24
of it together: 78 · 2.5 · 2^-24 = 2^-16.4 of the exponential; the polynomial is off by 2^-20,
reciprocal, exponential and products by 2^-22 or so. 2^-15 of the terms |f| (y) and
|Phi| + |x phi| and the like (dx) covers them twice over.
"""

from __future__ import annotations

import pytest
import torch

import sparsecore_amd as slk

pytestmark = pytest.mark.gpu


def normal(z):
    return 0.5 * torch.erfc(-z * 0.5 ** 0.5)


def bell(z):
    return torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5


def gelu(z):
    return z * normal(z), (normal(z), z * bell(z))


def silu(z):
    s = 1 / (1 + torch.exp(-z))
    return z * s, (s, z * s * (torch.exp(-z) * s))


def gelu_tanh(z):
    c = (2 / torch.pi) ** 0.5
    u2 = 2 * c * (z + 0.044715 * z ** 3)
    s = 1 / (1 + torch.exp(-u2))
    return z * s, (s, z * 2 * c * (1 + 3 * 0.044715 * z * z) * s * (torch.exp(-u2) * s))


# gelu_tanh's u is itself rounded three times: its argument doubles the count above, 2^-14
@pytest.mark.parametrize("f,lo,share", [(gelu, -12.5, 2.0 ** -15), (silu, -78.0, 2.0 ** -15),
                                        (gelu_tanh, -9.5, 2.0 ** -14)])
def test_bfloat16_tails(dev, f, lo, share):
    x = torch.linspace(lo, 3.0, 1 << 16, device=dev).bfloat16().requires_grad_()
    y = slk.activation(x, f.__name__, save_bits=32)
    dx, = torch.autograd.grad(y, [x], [torch.ones_like(y)])
    z = x.detach().double().cpu()
    want, (a, b) = f(z)
    half = torch.finfo(torch.bfloat16).eps / 2
    for name, got, exact, terms in (("y", y, want, want.abs()),
                                    ("dx", dx, a + b, a.abs() + b.abs())):
        off = (got.detach().double().cpu() - exact).abs() - (half * exact.abs() + share * terms)
        worst = int(off.argmax())
        assert float(off.max()) <= 1e-40, (name, float(z[worst]), float(off[worst]),
                                           float(exact[worst]))
