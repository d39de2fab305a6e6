"""sparsecore_amd.loss — the language-model head and its cross entropy as one operator.

    z = hidden · weightᵀ,    loss = logsumexp(z) - z[target]

without storing the logits: forward keeps a maximum and a sum of each token, backward
computes the logits again a piece of the vocabulary at a time (``slk_linear_ce_*``). Only
those of few tokens (at most 64 a row of the head) or of a small vocabulary (at most 128 a
token) are kept.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["linear_cross_entropy"]


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction, grad):
        d, v = weight.shape[1], weight.shape[0]
        n = target.numel()
        dev = hidden.device
        h, w, t = (x if x.is_contiguous() else x.contiguous() for x in (hidden, weight, target))
        keep = grad and any(ctx.needs_input_grad)
        loss = torch.empty(target.shape if reduction == "none" else (), device=dev)
        p = _lib.ptr
        args = _lib.LinearCE(n=n, d=d, v=v, ignore_index=ignore_index, hidden=p(h), weight=p(w),
                             target=p(t), loss=p(loss), dtype=_lib.DTYPES[h.dtype],
                             reduction=_lib.REDUCTIONS[reduction], keep=int(keep))
        saved = None
        if n == 0:
            loss.fill_(float("nan") if reduction == "mean" else 0.0)
        else:
            args.saved_bytes = _lib.linear_ce_saved_bytes(args)
            args.scratch_bytes = _lib.linear_ce_scratch_bytes(args, False)
            saved = torch.empty(args.saved_bytes, dtype=torch.uint8, device=dev) \
                if args.saved_bytes else None
            scratch = torch.empty(args.scratch_bytes, dtype=torch.uint8, device=dev)
            args.saved, args.scratch = p(saved), p(scratch)
            with _lib.on_device(h):
                _lib.linear_ce_forward(args, _lib.stream_of(h))
        if keep:
            ctx.save_for_backward(saved, h, w, t)
            ctx.rest = (n, d, v, ignore_index, reduction, hidden.shape, hidden.dtype)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        saved, h, w, t = ctx.saved_tensors
        n, d, v, ignore_index, reduction, shape, dtype = ctx.rest
        dev = grad.device
        dh = torch.empty(shape, dtype=dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            dw = (torch.empty if n else torch.zeros)((v, d), dtype=dtype, device=dev)
        if n:
            p = _lib.ptr
            up = grad.contiguous()
            args = _lib.LinearCE(n=n, d=d, v=v, ignore_index=ignore_index, hidden=p(h),
                                 weight=p(w), target=p(t), upstream=p(up), dhidden=p(dh), dweight=p(dw), saved=p(saved),
                                 saved_bytes=saved.numel(), dtype=_lib.DTYPES[dtype],
                                 reduction=_lib.REDUCTIONS[reduction], keep=1)
            args.scratch_bytes = _lib.linear_ce_scratch_bytes(args, True)
            scratch = torch.empty(args.scratch_bytes, dtype=torch.uint8, device=dev)
            args.scratch = p(scratch)
            with _lib.on_device(up):
                _lib.linear_ce_backward(args, _lib.stream_of(up))
        return dh, dw, None, None, None, None


def linear_cross_entropy(hidden, weight, target, *, ignore_index: int = -100,
                         reduction: str = "mean"):
    """Cross entropy of hidden · weightᵀ against target, logits never stored.

    Args:
        hidden: (..., D) hidden states, float32 or bfloat16.
        weight: (V, D) rows of the head, hidden's dtype.
        target: (...) int64 classes. A token with ``ignore_index`` has loss 0 and no
            gradient, and its hidden state reaches nothing, whatever it holds. Any other
            target outside [0, V) makes its loss NaN.
        reduction: "mean" (over the tokens not ignored; NaN if all are), "sum", or
            "none" (a loss per token, in target's shape).

    Returns the float32 loss, with gradients for hidden and weight. float32 products are
    about as exact as float32 matrix products, measured row by row: an element of hidden
    or weight keeps 22 bits down to 2^-39 of the largest in its row, a token's (a class's)
    terms of the gradient down to 2^-39 of its own largest. bfloat16 gradients pass
    through logit gradients rounded to bfloat16 where there are many. A forward that a backward may
    follow keeps weight and hidden once more, packed, until then; with few tokens (at most
    64, 32 in bfloat16) or a small vocabulary (128) the logits instead. hidden, weight and
    target must not change in place before the backward, whose scratch holds the logit
    gradients of a piece of the vocabulary: at most 512 MiB (twice that in float32), or 256
    rows over all tokens where those take more. Results repeat bit for bit.

    Raises TypeError (not a tensor), RuntimeError (not on the HIP device) and ValueError
    (shape, dtype, reduction).
    """
    for name, t in (("hidden", hidden), ("weight", weight), ("target", target)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"linear_cross_entropy: {name} must be a torch.Tensor, got "
                            f"{type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"linear_cross_entropy: {name} must be on a HIP (ROCm) device "
                               f"(got device={t.device})")
        if t.device != hidden.device:
            raise RuntimeError(f"linear_cross_entropy: {name} is on {t.device} but hidden on "
                               f"{hidden.device}")
    if reduction not in _lib.REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be one of "
                         f"{sorted(_lib.REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"linear_cross_entropy: weight must be (V, D), got "
                         f"{tuple(weight.shape)}")
    if hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] \
            or hidden.shape[:-1] != target.shape:
        raise ValueError(f"linear_cross_entropy: hidden {tuple(hidden.shape)}, weight "
                         f"{tuple(weight.shape)} and target {tuple(target.shape)} must be "
                         f"(..., D), (V, D) and (...)")
    if hidden.dtype not in _lib.DTYPES or weight.dtype != hidden.dtype:
        raise ValueError(f"linear_cross_entropy: hidden and weight must both be float32 or both "
                         f"bfloat16, got {hidden.dtype} and {weight.dtype}")
    if target.dtype != torch.int64:
        raise ValueError(f"linear_cross_entropy: target must be int64, got {target.dtype}")
    return _LinearCrossEntropy.apply(hidden, weight, target, int(ignore_index), reduction,
                                     torch.is_grad_enabled())
