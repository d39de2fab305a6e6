"""attention writes inside its arrays: outputs, gradients, saved and scratch memory of exactly
the size asked for, with guards around them, and gaps between strided rows left alone."""

from __future__ import annotations

import ctypes

import pytest
import torch

from sparsecore_amd import _lib
from sparsecore_amd.attn import _starts

pytestmark = pytest.mark.gpu

GUARD = 4096


class Guarded:
    """Memory of `nbytes` between two pieces of a known pattern."""

    def __init__(self, nbytes, dev):
        self.all = torch.full((nbytes + 2 * GUARD,), 0x5a, dtype=torch.uint8, device=dev)
        self.n = nbytes

    @property
    def ptr(self):
        return self.all.data_ptr() + GUARD

    def inside(self, dtype):
        return self.all[GUARD:GUARD + self.n].view(dtype)

    def whole(self):
        a = self.all
        return bool((a[:GUARD] == 0x5a).all()) and bool((a[GUARD + self.n:] == 0x5a).all())


def tensor(t, p=None):
    return _lib.AttnTensor(p or t.data_ptr(), *((0,) if t.dim() == 3 else ()), *t.stride())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode,h,g,d,n,tq,tk", [
    ("batch", 4, 2, 64, 2, 150, 150), ("batch", 4, 1, 128, 1, 65, 700),
    ("batch", 2, 2, 40, 3, 1, 129), ("lengths", 3, 3, 32, 4, 140, 140),
    ("packed", 8, 2, 128, 6, 500, 500), ("packed", 2, 1, 33, 40, 333, 333)])
def test_guards(dev, dtype, mode, h, g, d, n, tq, tk):
    lead = (n,) if mode != "packed" else ()
    shapes = {"q": (*lead, tq, h, d), "k": (*lead, tk, g, d), "v": (*lead, tk, g, d),
              "dout": (*lead, tq, h, d)}
    gen = torch.Generator().manual_seed(0)
    x = {k: torch.randn(*s, generator=gen).to(dtype).to(dev) for k, s in shapes.items()}
    bias = torch.randn(16, h, generator=gen).to(dev)
    dbias = Guarded(bias.numel() * 4, dev)
    elem = x["q"].element_size()
    # rows three elements apart: the gaps are nobody's
    gap = 3
    outs = {}
    for name, like in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v")):
        s = shapes[like]
        rows, width = s[-3] * (s[0] if lead else 1), s[-2] * s[-1]
        mem = Guarded(rows * (width + gap) * elem, dev)
        stride = (width + gap, s[-1], 1)
        if lead:
            stride = (s[-3] * (width + gap), *stride)
        outs[name] = (mem, s, stride)
    starts = _starts(16, 64)
    a = _lib.Attention(n=n, rows_q=tq, rows_k=tk, heads=h, kv_heads=g, dim=d, scale=d ** -0.5,
                       dtype=_lib.DTYPES[dtype], causal=1, keep=1, bias=bias.data_ptr(),
                       bias_dtype=0, buckets=16, max_distance=64,
                       bucket_starts=ctypes.addressof(starts), dbias=dbias.ptr,
                       **{k: tensor(t) for k, t in x.items()})
    for name, (mem, s, stride) in outs.items():
        setattr(a, name, _lib.AttnTensor(mem.ptr, *((0,) if len(s) == 3 else ()), *stride))
    ints = None
    if mode == "packed":
        ints = torch.linspace(2, tq - 1, n + 1).int().to(dev)
        a.q_offsets = ints.data_ptr()
    elif mode == "lengths":
        ints = torch.tensor([tq, 1, 0, tq // 2], dtype=torch.int32, device=dev)
        a.q_lengths = a.k_lengths = ints.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    results = []
    for keep in (0, 1):
        a.keep = keep
        a.saved_bytes = _lib.attention_saved_bytes(a)
        saved = Guarded(a.saved_bytes, dev)
        a.saved = saved.ptr
        a.scratch_bytes = _lib.attention_scratch_bytes(a, False)
        scratch = Guarded(a.scratch_bytes, dev)
        a.scratch = scratch.ptr
        _lib.attention_forward(a, stream)
        torch.cuda.synchronize()
        assert saved.whole() and scratch.whole() and outs["out"][0].whole()
        results.append(outs["out"][0].inside(dtype).clone())
    a.scratch_bytes = _lib.attention_scratch_bytes(a, True)
    back = Guarded(a.scratch_bytes, dev)
    a.scratch = back.ptr
    _lib.attention_backward(a, stream)
    torch.cuda.synchronize()
    assert saved.whole() and back.whole() and dbias.whole()
    assert dbias.inside(torch.float32).isfinite().all()
    for name, (mem, s, stride) in outs.items():
        assert mem.whole(), name
        rows, width = s[-3] * (s[0] if lead else 1), s[-2] * s[-1]
        flat = mem.inside(dtype).view(rows, width + gap)
        pattern = torch.full((gap * elem,), 0x5a, dtype=torch.uint8, device=dev).view(dtype)
        assert (flat[:, width:].contiguous().view(torch.uint8)
                == pattern.view(torch.uint8)).all(), name
        assert flat[:, :width].isfinite().all(), name
