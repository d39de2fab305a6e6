"""sparsecore_amd.act — activations whose backward pass needs a byte an element.

    y = f(x),    dx = dy · f'(x~)

in one pass each way (``slk_activation_*``). Between forward and backward x is kept in 8
bits: 256 consecutive elements of its memory share a float32 scale, the largest magnitude
`top` among them, and x~ is the nearest multiple of top / 127. ``SparseLinear(...,
save_bits=8)`` keeps its input in the same way.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["activation"]


@functools.lru_cache(maxsize=256)
def _fills(shape, stride) -> bool:
    want = 1
    for size, step in sorted(((n, s) for n, s in zip(shape, stride) if n != 1),
                             key=lambda x: x[1]):
        if step != want:
            return False
        want *= size
    return True


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one piece of memory, in any order of its dimensions."""
    return t.is_contiguous() or _fills(t.shape, t.stride())


def _in_layout(t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    """t in the memory order of like, which is dense."""
    if t.stride() == like.stride():
        return t
    if t.dim() == 2 and t.dtype == torch.float32:
        from .ops import _as_row_major

        return _as_row_major(t) if like.is_contiguous() else _as_row_major(t.t()).t()
    return torch.empty_like(like).copy_(t)


def encode8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of a dense float32 or bfloat16 x, in its memory order."""
    n = x.numel()
    codes = torch.empty(n, dtype=torch.int8, device=x.device)
    scales = torch.empty(-(-n // _lib.ACT_BLOCK), device=x.device)
    p = _lib.ptr
    with _lib.on_device(x):
        _lib.activation_forward(
            _lib.Activation(n=n, x=p(x), codes=p(codes), scales=p(scales),
                            dtype=_lib.DTYPES[x.dtype], kind=0), _lib.stream_of(x))
    return codes, scales


def decode8(codes: torch.Tensor, scales: torch.Tensor, shape) -> torch.Tensor:
    """The float32 values that codes stand for, contiguous, of the given shape."""
    out = torch.empty(shape, device=codes.device)
    p = _lib.ptr
    with _lib.on_device(codes):
        _lib.activation_backward(
            _lib.Activation(n=codes.numel(), dx=p(out), codes=p(codes), scales=p(scales),
                            dtype=_lib.SLK_F32, kind=0), _lib.stream_of(codes))
    return out


class _Activation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind, save_bits, grad):
        if not _dense(x):
            x = x.contiguous()
        n, dev = x.numel(), x.device
        y = torch.empty_like(x)
        p = _lib.ptr
        args = _lib.Activation(n=n, x=p(x), y=p(y), dtype=_lib.DTYPES[x.dtype], kind=kind)
        keep = grad and ctx.needs_input_grad[0]
        codes = scales = None
        if keep and save_bits == 8:
            codes = torch.empty(n, dtype=torch.int8, device=dev)
            scales = torch.empty(-(-n // _lib.ACT_BLOCK), device=dev)
            args.codes, args.scales = p(codes), p(scales)
        with _lib.on_device(x):
            _lib.activation_forward(args, _lib.stream_of(x))
        if keep:
            ctx.save_for_backward(codes, scales, x if save_bits == 32 else None)
            ctx.rest = (kind, x.shape, x.stride(), x.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales, x = ctx.saved_tensors
        kind, shape, stride, dtype = ctx.rest
        dx = torch.empty_strided(shape, stride, dtype=dtype, device=dy.device)
        dy = _in_layout(dy, dx)
        p = _lib.ptr
        args = _lib.Activation(n=dx.numel(), x=p(x), dy=p(dy), dx=p(dx), codes=p(codes),
                               scales=p(scales), dtype=_lib.DTYPES[dtype], kind=kind)
        with _lib.on_device(dy):
            _lib.activation_backward(args, _lib.stream_of(dy))
        return dx, None, None, None


def activation(x, kind: str = "gelu", *, save_bits: int = 8):
    """f(x) with f's gradient taken at x as 8 bits keep it, autograd-aware.

    Args:
        x: float32 or bfloat16, any shape; y has x's memory layout (a feature-major view, as
            a SparseLinear returns it, stays one).
        kind: "gelu" (exact), "gelu_tanh" (its tanh form), "silu" or "relu".
        save_bits: 8, or 32 to keep x itself for the backward (no rounding).

    y is computed from x itself; only the backward reads the codes. A block of 256
    consecutive elements of x's memory shares the scale `top`, its largest finite magnitude:
    the kept x is off by at most top / 254, blocks below 2^-100 are kept as zeros, and an
    element that is not finite is kept as NaN without touching its neighbours. relu's slope
    is that of the kept value: 0 where it is 0. Arithmetic is float32, rounded once.

    Raises TypeError (not a tensor), RuntimeError (not on the HIP device) and ValueError
    (dtype, kind, save_bits).
    """
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"activation: x must be a torch.Tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise RuntimeError(f"activation: x must be on a HIP (ROCm) device (got "
                           f"device={x.device})")
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"activation: x must be float32 or bfloat16, got {x.dtype}")
    code = _lib.ACT_KINDS.get(kind)
    if not code:
        raise ValueError(f"activation: kind must be one of "
                         f"{sorted(set(_lib.ACT_KINDS) - {'none'})}, got {kind!r}")
    if save_bits not in (8, 32):
        raise ValueError(f"activation: save_bits must be 8 or 32, got {save_bits}")
    return _Activation.apply(x, code, save_bits, torch.is_grad_enabled())
