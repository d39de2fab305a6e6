"""sparsecore_amd.norm — what stands between two blocks of a model, as one operator:

    r = x + scale · gate ∘ post(branch),    y = pre(r)

the residual sum of a block's output (through an optional norm of its own and an
optional gate) and the norm before the next block, forward and backward in one pass
over the arrays each (``slk_norm_forward``, ``slk_norm_backward``).

A SparseLinear returns its output, and takes its input without a copy, feature by
feature in memory (the transposed view of a feature-major array). ``branch`` and the
gradient of ``y`` are read in either layout, and ``feature_major=True`` writes ``y`` so,
so that a block's norm, sparse layers and residual need no transposing copies.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["residual_norm", "ResidualNorm"]

_KINDS = {"layer": 1, "rms": 0}


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """A contiguous N x D copy of a feature-major view (t itself if contiguous)."""
    from .ops import _as_row_major

    return _as_row_major(t) if t.dtype == torch.float32 else t.contiguous()


def _as_cols(t: torch.Tensor) -> torch.Tensor:
    """The same N x D values, feature by feature in memory."""
    return _as_rows(t.t()).t()


def _layout(t: torch.Tensor, n: int, d: int) -> tuple[torch.Tensor, int]:
    """(N x D tensor, 1 if it is feature-major): a layout that the kernels read."""
    if t.is_contiguous():
        return t, 0
    if t.dim() != 2:
        t = t.reshape(n, d)
    if t.stride(0) == 1 and t.stride(1) == n:
        return (t, 1) if d <= _lib.NORM_COLS_MAX else (_as_rows(t), 0)
    return t.contiguous(), 0


def _packed(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _gate_rows(gate: torch.Tensor, x: torch.Tensor, n: int, d: int) -> int:
    """Rows of gate over x's tokens, in order; ValueError for any other shape."""
    if gate.shape == (d,):
        return 1
    if gate.shape == x.shape:
        return n
    if x.dim() == 2 and gate.dim() == 2 and gate.shape[1] == d and gate.shape[0] > 0 \
            and n % gate.shape[0] == 0:
        return gate.shape[0]
    if x.dim() > 2 and gate.dim() == x.dim() and gate.shape[-1] == d:
        lead = list(gate.shape[:-1])
        k = len(lead)
        while k and lead[k - 1] == 1:
            k -= 1
        if lead[:k] == list(x.shape[:k]):
            return gate.numel() // d
    raise ValueError(f"residual_norm: gate of shape {tuple(gate.shape)} does not fit x of shape "
                     f"{tuple(x.shape)}: (D,), x's shape, x's leading sizes then ones, or for a "
                     f"2-D x (G, D) with G dividing N")


class _ResidualNorm(torch.autograd.Function):
    """Outputs (r, y), or y alone where there is no branch."""

    @staticmethod
    def forward(ctx, x, weight, bias, branch, gate, post_weight, post_bias, scale, layer, eps,
                feature_major, grad):
        # Small calls are bound by this host work: as few tensor operations as possible.
        shape, dt, dev = x.shape, x.dtype, x.device
        d = shape[-1]
        n = x.numel() // d
        x = _packed(x)
        u, u_cols = _layout(branch, n, d) if branch is not None else (None, 0)
        rows = _gate_rows(gate, x, n, d) if gate is not None else 0
        weight, bias, gate = _packed(weight), _packed(bias), _packed(gate)
        post_weight, post_bias = _packed(post_weight), _packed(post_bias)
        y_cols = int(feature_major and d <= _lib.NORM_COLS_MAX)
        if y_cols:
            y = torch.empty((d, n), dtype=dt, device=dev).t()
            if len(shape) != 2:
                y = y.reshape(shape)
        else:
            y = torch.empty(shape, dtype=dt, device=dev)
        r = torch.empty(shape, dtype=dt, device=dev) if u is not None else x
        need = ctx.needs_input_grad
        stats = torch.empty((n, 4), device=dev) if grad and any(need) else None
        if n:
            p = _lib.ptr
            args = _lib.Norm(n=n, d=d, gate_rows=rows, x=p(x), branch=p(u), gate=p(gate),
                             weight=p(weight), bias=p(bias), post_weight=p(post_weight),
                             post_bias=p(post_bias), r=p(r), y=p(y), stats=p(stats), scale=scale,
                             eps=eps, dtype=_lib.DTYPES[dt], layer=layer, branch_cols=u_cols,
                             y_cols=y_cols)
            with _lib.on_device(x):
                _lib.norm_forward(args, _lib.stream_of(x))
        if feature_major and not y_cols:
            y = _as_cols(y.reshape(n, d)).reshape(shape)
        if stats is not None:
            ctx.set_materialize_grads(False)
            keep_u = post_weight is not None or (gate is not None and need[4])
            ctx.save_for_backward(r, stats, weight, bias, u if keep_u else None, gate,
                                  post_weight, post_bias)
            # the branch's gradient goes back in the branch's layout
            back_cols = (u is not None and not u_cols and n > 1 and d > 1
                         and not branch.is_contiguous()
                         and branch.reshape(n, d).t().is_contiguous())
            ctx.rest = (shape, n, d, rows, scale, layer, eps, u_cols, back_cols,
                        branch is not None)
        return (r, y) if branch is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        r, stats, weight, bias, u, gate, post_weight, post_bias = ctx.saved_tensors
        shape, n, d, rows, scale, layer, eps, u_cols, back_cols, has_branch = ctx.rest
        need = ctx.needs_input_grad
        dr, dy = grads if has_branch else (None, grads[0])
        dt, dev = r.dtype, r.device
        y_cols = 0
        if dr is not None and not dr.is_contiguous():
            dr = _as_rows(dr.reshape(n, d))
        if dy is not None:
            dy, y_cols = _layout(dy, n, d)

        dx = torch.empty(shape, dtype=dt, device=dev) if need[0] else None
        du = None
        if has_branch and need[3]:
            if u_cols:
                du = torch.empty((d, n), dtype=dt, device=dev).t()
                if len(shape) != 2:
                    du = du.reshape(shape)
            else:
                du = torch.empty(shape, dtype=dt, device=dev)
        dgate = None
        if gate is not None and need[4]:
            dgate = (torch.zeros if n == 0 else torch.empty)(gate.shape, dtype=dt, device=dev)
        # weight's, bias's, post_weight's and post_bias's gradients; without dy there is
        # nothing to sum for the first two, without tokens for any
        wanted = [(need[1], dy is None), (need[2] and bias is not None, dy is None),
                  (need[5] and post_weight is not None, False),
                  (need[6] and post_bias is not None, False)]
        sums = [None] * 4
        for k, (want, empty) in enumerate(wanted):
            if want:
                sums[k] = (torch.zeros if empty or n == 0 else torch.empty)(d, dtype=dt,
                                                                           device=dev)
        if n:
            p = _lib.ptr
            # where the branch itself is not needed any address stands for it (not read)
            branch = p(u) if u is not None else (p(r) if has_branch else None)
            args = _lib.Norm(n=n, d=d, gate_rows=rows, branch=branch, gate=p(gate),
                             weight=p(weight), bias=p(bias), post_weight=p(post_weight),
                             post_bias=p(post_bias), r=p(r), stats=p(stats), dr=p(dr), dy=p(dy),
                             dx=p(dx), dbranch=p(du), dgate=p(dgate), dweight=p(sums[0]),
                             dbias=p(sums[1]), dpost_weight=p(sums[2]), dpost_bias=p(sums[3]),
                             scale=scale, eps=eps, dtype=_lib.DTYPES[dt], layer=layer,
                             branch_cols=u_cols, y_cols=y_cols)
            nbytes = _lib.norm_workspace_bytes(args)
            if nbytes:
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
                args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
            with _lib.on_device(r):
                _lib.norm_backward(args, _lib.stream_of(r))
            if du is not None and back_cols:
                du = _as_cols(du.reshape(n, d)).reshape(shape)
        return (dx, sums[0], sums[1], du, dgate, sums[2], sums[3], None, None, None, None, None)


def residual_norm(x, weight, bias=None, *, branch=None, gate=None, post_weight=None,
                  post_bias=None, scale: float = 1.0, kind: str = "layer", eps: float = 1e-5,
                  feature_major: bool = False):
    """(r, y) with r = x + scale · gate ∘ post(branch) and y = pre(r), autograd-aware.

    Args:
        x: the residual stream, (..., D), float32 or bfloat16, D <= 16384.
        weight, bias: of the norm before the next block, (D,); bias optional.
        branch: the block's output, x's shape, token-major or the transposed view of a
            feature-major array. None: r is x itself.
        gate: scales the branch: (D,) for all tokens alike, x's shape, or x's leading
            sizes followed by ones, as (B, 1, D) for a gate of each sequence. For a 2-D x
            also (G, D): row i serves the i-th N/G consecutive tokens.
        post_weight, post_bias: of a norm of the branch itself, (D,).
        scale: constant factor of the branch.
        kind: "layer" (LayerNorm) or "rms" (RMSNorm, which has no biases), of both norms.
        feature_major: write y feature by feature in memory (y is a transposed view), as
            a SparseLinear takes it without a copy.

    All tensors share x's dtype; arithmetic, means and sums are float32, and y is
    computed from the unrounded r. The backward reads r as it was returned, so in
    bfloat16 its normalised values carry r's rounding (2^-9 of r, about 1.4 times the
    error of gradients from an unrounded r), with the forward's own mean and deviation.
    Every gradient is computed in one pass and repeats bit for bit.

    Raises TypeError (not a tensor), RuntimeError (not on the HIP device) and ValueError
    (shape, dtype, kind).
    """
    if kind not in _KINDS:
        raise ValueError(f"residual_norm: kind must be 'layer' or 'rms', got {kind!r}")
    given = [("x", x), ("weight", weight), ("bias", bias), ("branch", branch), ("gate", gate),
             ("post_weight", post_weight), ("post_bias", post_bias)]
    for name, t in given:
        if t is None and name not in ("x", "weight"):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"residual_norm: {name} must be a torch.Tensor, got "
                            f"{type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"residual_norm: {name} must be on a HIP (ROCm) device (got "
                               f"device={t.device})")
        if t.device != x.device:
            raise RuntimeError(f"residual_norm: {name} is on {t.device} but x on {x.device}")
        if t.dtype != x.dtype:
            raise ValueError(f"residual_norm: {name} is {t.dtype} but x is {x.dtype}")
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"residual_norm: x must be float32 or bfloat16, got {x.dtype}")
    d = x.shape[-1] if x.dim() else 0
    if not 1 <= d <= _lib.NORM_MAX_D:
        raise ValueError(f"residual_norm: x must have between 1 and {_lib.NORM_MAX_D} features, "
                         f"got shape {tuple(x.shape)}")
    for name, t in given[1:]:
        if t is not None and name not in ("branch", "gate") and t.shape != (d,):
            raise ValueError(f"residual_norm: {name} must have shape ({d},), got "
                             f"{tuple(t.shape)}")
    if branch is None:
        if gate is not None or post_weight is not None:
            raise ValueError("residual_norm: a gate or a post norm needs a branch")
    elif branch.shape != x.shape:
        raise ValueError(f"residual_norm: branch has shape {tuple(branch.shape)} but x "
                         f"{tuple(x.shape)}")
    if post_bias is not None and post_weight is None:
        raise ValueError("residual_norm: post_bias needs post_weight")
    if kind == "rms" and (bias is not None or post_bias is not None):
        raise ValueError("residual_norm: RMSNorm has no bias")
    if gate is not None:
        _gate_rows(gate, x, x.numel() // d, d)
    out = _ResidualNorm.apply(x, weight, bias, branch, gate, post_weight, post_bias,
                              float(scale), _KINDS[kind], float(eps), bool(feature_major),
                              torch.is_grad_enabled())
    return out if branch is not None else (x, out)


class ResidualNorm(nn.Module):
    """The residual sum of a block and the norm before the next one, with its parameters.

    ``r, y = norm(x, branch)``: r = x + scale · gate ∘ post(branch), y = pre(r); with no
    branch yet, ``r`` is ``x``.

    Args:
        d: features.
        kind: "layer" or "rms".
        post: norm the branch too, with a weight (and bias) of its own.
        gate: learn a gate of each feature, initialised to this value (None: none).
        scale: constant factor of the branch.
        bias: biases of a LayerNorm.
        feature_major: write y as a SparseLinear takes it without a copy.
    """

    def __init__(self, d: int, kind: str = "layer", *, post: bool = False,
                 gate: float | None = None, scale: float = 1.0, eps: float = 1e-5,
                 bias: bool = True, feature_major: bool = True, device=None, dtype=None):
        super().__init__()
        if kind not in _KINDS:
            raise ValueError(f"ResidualNorm: kind must be 'layer' or 'rms', got {kind!r}")
        self.d, self.kind, self.scale, self.eps = d, kind, scale, eps
        self.feature_major = feature_major
        make = dict(device=device, dtype=dtype)
        bias = bias and kind == "layer"

        def vector(value, wanted):
            return nn.Parameter(torch.full((d,), float(value), **make)) if wanted else None

        self.weight, self.bias = vector(1.0, True), vector(0.0, bias)
        self.post_weight, self.post_bias = vector(1.0, post), vector(0.0, post and bias)
        self.gate = vector(0.0 if gate is None else gate, gate is not None)

    def forward(self, x, branch=None):
        if branch is None:
            return residual_norm(x, self.weight, self.bias, kind=self.kind, eps=self.eps,
                                 feature_major=self.feature_major)
        return residual_norm(x, self.weight, self.bias, branch=branch, gate=self.gate,
                             post_weight=self.post_weight, post_bias=self.post_bias,
                             scale=self.scale, kind=self.kind, eps=self.eps,
                             feature_major=self.feature_major)

    def extra_repr(self) -> str:
        return (f"{self.d}, kind={self.kind!r}, post={self.post_weight is not None}, "
                f"gate={self.gate is not None}, scale={self.scale}")
