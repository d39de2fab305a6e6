"""sparsecore_amd.attn — attention between two projections of a model:

    S = scale · Q·Kᵀ (+ bias of the distance),   P = softmax(S),   out = P·V

forward and backward, scores never stored (``slk_attention_*``): a batch, a padded batch
or packed sequences, grouped heads, causal or not, with a learned bias of the relative
position.

A SparseLinear returns its output feature by feature in memory (the transposed view of a
feature-major array). Queries, keys, values and the output's gradient are read with any
strides, gradients come back in their tensors' layout, and ``feature_major=True`` writes
the output as the next SparseLinear takes it without a copy.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["attention", "relative_buckets"]


@functools.lru_cache(maxsize=64)
def relative_buckets(buckets: int, max_distance: int) -> tuple[int, ...]:
    """First distance of each of one side's buckets: the first half hold one distance each
    (0, 1, ...), the others grow by a constant factor up to ``max_distance``, where the last
    one would end. With e of the first kind and r = buckets - e, bucket e + t begins at the
    first n with (n / e)^r >= (max_distance / e)^t, decided in whole numbers."""
    if buckets < 2:
        raise ValueError(f"relative_buckets: at least 2 buckets a side, got {buckets}")
    e = buckets // 2
    r = buckets - e
    if max_distance <= e:
        raise ValueError(f"relative_buckets: max_distance must be above {e}, got {max_distance}")
    starts = list(range(e + 1))
    n = e
    for t in range(1, r):
        bar = e ** (r - t) * max_distance ** t
        while n ** r < bar:
            n += 1
        starts.append(n)
    return tuple(starts[:buckets])


@functools.lru_cache(maxsize=64)
def _starts(buckets: int, max_distance: int):
    table = relative_buckets(buckets, max_distance)
    return (ctypes.c_int32 * len(table))(*table)


def _tensor(t: torch.Tensor) -> _lib.AttnTensor:
    if t.dim() == 3:
        return _lib.AttnTensor(t.data_ptr(), 0, *t.stride())
    return _lib.AttnTensor(t.data_ptr(), *t.stride())


@functools.lru_cache(maxsize=256)
def _compact(shape, stride) -> tuple[int, ...]:
    """Strides of a tensor of this shape in the same order of dimensions, without gaps."""
    out, step = [0] * len(shape), 1
    for i in sorted(range(len(shape)), key=lambda i: (stride[i], -i)):
        out[i] = step
        step *= shape[i]
    return tuple(out)


def _gradient(like, dtype, device) -> tuple[torch.Tensor, _lib.AttnTensor]:
    """A new tensor for the gradient of one of this shape and these strides."""
    shape, stride = like
    stride = _compact(shape, stride)
    t = torch.empty_strided(shape, stride, dtype=dtype, device=device)
    return t, _lib.AttnTensor(t.data_ptr(), *((0,) if len(shape) == 3 else ()), *stride)


def _output(q: torch.Tensor, feature_major: bool) -> torch.Tensor:
    if not feature_major:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    *lead, h, d = q.shape
    rows = lead[0] * lead[1] if len(lead) == 2 else lead[0]
    stride = (d * rows, rows) if rows else (d, 1)
    return torch.empty_strided(q.shape, ((lead[1], 1) if len(lead) == 2 else (1,)) + stride,
                               dtype=q.dtype, device=q.device)


def _set_ints(a, offsets, k_offsets, lengths, k_lengths) -> None:
    p = _lib.ptr
    a.q_offsets, a.k_offsets = p(offsets), p(k_offsets)
    a.q_lengths, a.k_lengths = p(lengths), p(k_lengths)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, offsets, k_offsets, lengths, k_lengths, max_distance, causal,
                scale, feature_major, grad):
        # Small calls are bound by this host work: as few tensor operations as possible.
        dev = q.device
        keep = grad and any(ctx.needs_input_grad)
        out = _output(q, feature_major)
        a = _lib.Attention(
            n=offsets.shape[0] - 1 if offsets is not None else q.shape[0], rows_q=q.shape[-3],
            rows_k=k.shape[-3], heads=q.shape[-2], kv_heads=k.shape[-2], dim=q.shape[-1],
            q=_tensor(q), k=_tensor(k), v=_tensor(v), out=_tensor(out), scale=scale,
            dtype=_lib.DTYPES[q.dtype], causal=causal, keep=keep)
        _set_ints(a, offsets, k_offsets, lengths, k_lengths)
        if bias is not None:
            if not bias.is_contiguous():
                bias = bias.contiguous()
            a.bias, a.bias_dtype = bias.data_ptr(), _lib.DTYPES[bias.dtype]
            a.buckets, a.max_distance = bias.shape[0], max_distance
            starts = _starts(bias.shape[0] if causal else bias.shape[0] // 2, max_distance)
            a.bucket_starts = ctypes.addressof(starts)
        saved = None
        with _lib.on_device(q):
            if keep:
                a.saved_bytes = _lib.attention_saved_bytes(a)
                saved = torch.empty(a.saved_bytes, dtype=torch.uint8, device=dev)
                a.saved = saved.data_ptr()
            a.scratch_bytes = _lib.attention_scratch_bytes(a, False)
            if a.scratch_bytes:
                scratch = torch.empty(a.scratch_bytes, dtype=torch.uint8, device=dev)
                a.scratch = scratch.data_ptr()
            _lib.attention_forward(a, _lib.stream_of(q))
        if keep:
            ctx.save_for_backward(saved, out, bias, offsets, k_offsets, lengths, k_lengths)
            ctx.args, ctx.starts = a, starts if bias is not None else None
            ctx.like = [(t.shape, t.stride()) for t in (q, k, v)]
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        saved, out, bias, *ints = ctx.saved_tensors
        need = ctx.needs_input_grad
        # a copy: the graph may be gone through again
        a = _lib.Attention.from_buffer_copy(ctx.args)
        _set_ints(a, *ints)
        dtype, dev = out.dtype, out.device
        dq = dk = dv = dbias = None
        if need[0]:
            dq, a.dq = _gradient(ctx.like[0], dtype, dev)
        if need[1] or need[2]:  # computed together
            dk, a.dk = _gradient(ctx.like[1], dtype, dev)
            dv, a.dv = _gradient(ctx.like[2], dtype, dev)
        if bias is not None:
            a.bias = bias.data_ptr()
            if need[3]:
                dbias = torch.empty_like(bias)
                a.dbias = dbias.data_ptr()
        a.out, a.dout, a.saved = _tensor(out), _tensor(dout), saved.data_ptr()
        with _lib.on_device(out):
            a.scratch_bytes = _lib.attention_scratch_bytes(a, True)
            if a.scratch_bytes:
                scratch = torch.empty(a.scratch_bytes, dtype=torch.uint8, device=dev)
                a.scratch = scratch.data_ptr()
            _lib.attention_backward(a, _lib.stream_of(out))
        return (dq, dk if need[1] else None, dv if need[2] else None, dbias) + (None,) * 9


def attention(q, k, v, *, causal: bool = True, scale: float | None = None, offsets=None,
              k_offsets=None, lengths=None, k_lengths=None, bias=None, max_distance: int = 128,
              feature_major: bool = False):
    """softmax(scale · q·kᵀ + bias) · v over the keys that each query sees, autograd-aware.

    Args:
        q: (B, T, H, D) queries, or (N, H, D) packed ones, float32 or bfloat16, D <= 128.
        k, v: (B, S, G, D) or (M, G, D) keys and values, q's dtype; G divides H, and key head
            i serves the query heads i·H/G .. (i + 1)·H/G - 1.
        causal: a sequence's last query stands at its last key: of n queries and m keys,
            query i sees the keys up to i + m - n. Else every query sees every key.
        scale: factor of the scores, 0 to 2e38; default D ** -0.5.
        offsets: (sequences + 1,) int32: packed sequence i is the rows offsets[i] to
            offsets[i + 1] of q, and of k and v unless k_offsets is given.
        lengths: (B,) int32: the first lengths[b] queries of entry b are live, and as many
            keys unless k_lengths is given. k_lengths alone: live keys, all queries live, as
            when new tokens meet arrays of keys that are only partly filled.
        bias: (buckets, H) learned bias of the relative position, float32 or q's dtype. With
            causal, of how far the key is behind; else the first half is for keys at or
            behind the query and the second half for those ahead. See relative_buckets.
        max_distance: distances from here on share the last bucket; at most 256.
        feature_major: write the output feature by feature in memory (a view whose features
            are rows), as a SparseLinear takes it without a copy.

    Returns q's shape. A query that sees no key has output 0 and no gradient, and so has a
    row that belongs to no sequence; of one that sees a single key only the value has a
    gradient; what is masked reaches nothing, whatever it holds. A row
    of q, k, v or of the output's gradient with a value that is not finite makes NaN of the
    results that its row has a part in (for few queries without gradients, of what the value
    itself reaches). Offsets and lengths are read on the device: those out of range, or
    offsets that fall, count as the nearest that do not.

    Products run on the matrix cores' float16 instructions, each block of 64 rows of a head
    scaled by a power of two of its own, or each row where the block's rows are more than
    2^14 apart (then 1.5 to 1.7 times the time). float32 operands go in two parts: an element
    is off by at most 2^-22 of itself or 2^-25 of the largest of its row, about float32's own
    rounding. bfloat16 ones are exact down to 2^-17 of that. Between the products weights and
    the scores' gradients are rounded to 22 bits (bfloat16: 11), or to 2^-32 of the largest
    of their row of results where that is more (in dv to 2^-39 of 1). Softmax and sums are
    float32, in a fixed order: results repeat bit for bit. A forward that a backward may follow keeps q, k and v once more,
    packed (not the tensors themselves), and the output, which must not change in place
    before the backward, nor may offsets and lengths; of a bfloat16 output also what its
    rounding took off, in two bytes an element.

    Raises TypeError (not a tensor), RuntimeError (not on the HIP device) and ValueError
    (shape, dtype, sizes).
    """
    for name, t in (("q", q), ("k", k), ("v", v), ("bias", bias), ("offsets", offsets),
                    ("k_offsets", k_offsets), ("lengths", lengths), ("k_lengths", k_lengths)):
        if t is None and name not in ("q", "k", "v"):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"attention: {name} must be a torch.Tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"attention: {name} must be on a HIP (ROCm) device (got "
                               f"device={t.device})")
        if t.get_device() != q.get_device():
            raise RuntimeError(f"attention: {name} is on {t.device} but q on {q.device}")
    if q.dtype not in _lib.DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"attention: q, k and v must all be float32 or all bfloat16, got "
                         f"{q.dtype}, {k.dtype} and {v.dtype}")
    packed = offsets is not None
    rank = 3 if packed else 4
    if q.dim() != rank or k.dim() != rank or v.shape != k.shape:
        raise ValueError(f"attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v "
                         f"{tuple(v.shape)} must be "
                         + ("(N, H, D), (M, G, D) and (M, G, D)" if packed else
                            "(B, T, H, D), (B, S, G, D) and (B, S, G, D)"))
    h, d = q.shape[-2:]
    g = k.shape[-2]
    if k.shape[-1] != d or not 1 <= d <= _lib.ATTN_MAX_DIM:
        raise ValueError(f"attention: q and k must share a head size of 1 to "
                         f"{_lib.ATTN_MAX_DIM}, got {d} and {k.shape[-1]}")
    if g < 1 or h < 1 or h % g:
        raise ValueError(f"attention: {h} query heads are no multiple of {g} key heads")
    if packed:
        if lengths is not None or k_lengths is not None:
            raise ValueError("attention: offsets or lengths, not both")
        if k_offsets is None and k.shape[0] != q.shape[0]:
            raise ValueError(f"attention: {q.shape[0]} query rows but {k.shape[0]} key rows "
                             f"share offsets")
    else:
        if k_offsets is not None:
            raise ValueError("attention: k_offsets need offsets")
        if q.shape[0] != k.shape[0]:
            raise ValueError(f"attention: q has {q.shape[0]} entries but k {k.shape[0]}")
    for name, t in (("offsets", offsets), ("k_offsets", k_offsets), ("lengths", lengths),
                    ("k_lengths", k_lengths)):
        if t is None:
            continue
        each = name.endswith("lengths")
        if t.dtype != torch.int32 or t.dim() != 1 or \
                (t.shape[0] != q.shape[0] if each else t.shape[0] < 1):
            raise ValueError(f"attention: {name} must be int32, one for each "
                             f"{'entry' if each else 'sequence and one more'}, got {t.dtype} "
                             f"{tuple(t.shape)}")
    if k_offsets is not None and k_offsets.shape != offsets.shape:
        raise ValueError("attention: offsets and k_offsets must have the same length")
    if lengths is not None and k_lengths is None:
        k_lengths = lengths
    if bias is not None:
        if bias.dim() != 2 or bias.shape[1] != h:
            raise ValueError(f"attention: bias must be (buckets, {h}), got {tuple(bias.shape)}")
        if bias.dtype not in (torch.float32, q.dtype):
            raise ValueError(f"attention: bias must be float32 or {q.dtype}, got {bias.dtype}")
        buckets = bias.shape[0]
        if not 2 <= (buckets if causal else buckets // 2) or \
                buckets > _lib.ATTN_MAX_BUCKETS or (not causal and buckets % 2):
            raise ValueError(f"attention: bias must have 2 to {_lib.ATTN_MAX_BUCKETS} buckets "
                             f"(causal), or an even number from 4 on, got {buckets}")
        max_distance = int(max_distance)
        if not 1 <= max_distance <= _lib.ATTN_MAX_DISTANCE:
            raise ValueError(f"attention: max_distance must be between 1 and "
                             f"{_lib.ATTN_MAX_DISTANCE}, got {max_distance}")
        _starts(buckets if causal else buckets // 2, max_distance)
    scale = d ** -0.5 if scale is None else float(scale)
    if not (0.0 <= scale < math.inf):
        raise ValueError(f"attention: scale must be finite and not negative, got {scale}")
    if offsets is not None or k_lengths is not None:
        offsets, k_offsets, lengths, k_lengths = (
            t if t is None or t.is_contiguous() else t.contiguous()
            for t in (offsets, k_offsets, lengths, k_lengths))
    return _Attention.apply(q, k, v, bias, offsets, k_offsets, lengths, k_lengths, max_distance,
                            bool(causal), scale, bool(feature_major), torch.is_grad_enabled())
