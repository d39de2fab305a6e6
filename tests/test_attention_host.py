"""attention and activation on the host: tensors off the GPU are refused, the C-ABI's checks
answer before any device work (fake, never dereferenced pointers), and the buckets of a
relative position bias."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import sparsecore_amd as slk
from sparsecore_amd import _lib
from sparsecore_amd.act import _dense
from sparsecore_amd.attn import _compact, relative_buckets


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 2, 32)
    with pytest.raises(RuntimeError, match="HIP"):
        slk.attention(q, q, q)
    with pytest.raises(TypeError, match="Tensor"):
        slk.attention(None, q, q)
    with pytest.raises(RuntimeError, match="HIP"):
        slk.activation(q)
    with pytest.raises(ValueError, match="save_bits"):
        slk.SparseLinear(4, 4, save_bits=16)


def refused(rc, *words):
    msg = _lib.load().slk_last_error().decode()
    assert rc == _lib.SLK_EINVAL and all(w in msg for w in words), msg


STARTS = (ctypes.c_int32 * 8)(0, 1, 2, 3, 4, 8, 16, 32)


def tensor(p=16, row=64, head=64, feature=1, batch=0):
    return _lib.AttnTensor(p, batch, row, head, feature)


def arguments(**kw):
    a = dict(n=2, rows_q=100, rows_k=100, heads=4, kv_heads=2, dim=64, scale=0.125, dtype=0,
             causal=1, keep=1, saved=16, saved_bytes=1 << 50, scratch=16, scratch_bytes=1 << 50)
    for k in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        a[k] = tensor()
    return _lib.Attention(**{**a, **kw})


@pytest.mark.parametrize("backward", [False, True])
def test_attention_checks_on_the_host(backward):
    lib = _lib.load()
    f = lib.slk_attention_backward if backward else lib.slk_attention_forward

    def no(*words, **kw):
        refused(f(ctypes.byref(arguments(**kw)), None), *words)

    refused(f(None, None), "NULL arguments")
    no("negative size", rows_q=-1)
    no("dtype", dtype=3)
    no("dim in [1", dim=0)
    no("dim in [1", dim=129)
    no("multiple of kv_heads", heads=3)
    no("multiple of kv_heads", kv_heads=0)
    no("multiple of kv_heads", heads=32768, kv_heads=1)
    no("scale", scale=-1.0)
    no("scale", scale=float("nan"))
    no("scale", scale=float("inf"))
    no("not both", q_offsets=16, q_lengths=16)
    no("k_offsets need", k_offsets=16)
    no("share offsets", q_offsets=16, rows_k=99)
    start = ctypes.addressof(STARTS)
    bias = dict(bias=16, buckets=8, max_distance=32, bucket_starts=start)
    no("bias dtype", **{**bias, "bias_dtype": 7})
    no("buckets", **{**bias, "buckets": 129})
    no("buckets", **{**bias, "buckets": 7, "causal": 0})
    no("max_distance", **{**bias, "max_distance": 257})
    no("begin with 0", **{**bias, "bucket_starts": None})
    no("ascend", **{**bias, "max_distance": 31})
    no("NULL out" if backward else "NULL q", **{("dout" if backward else "q"): tensor(None)})
    no("saved too small", saved_bytes=1000)
    no("saved too small", saved=None)
    no("scratch too small", **({"scratch_bytes": 1000} if backward else
                               {"scratch_bytes": 10, "keep": 0}))
    no("aligned", saved=24)
    no("too many rows", rows_q=1 << 31)
    no("too many rows", n=1 << 20, rows_q=1 << 12)
    no("too many", n=1 << 14, rows_q=1 << 15, heads=16384, kv_heads=1)
    if backward:
        no("go together", dk=tensor(None))
        no("without a bias", dbias=16)
    else:
        no("NULL k or v", k=tensor(None))
    assert f(ctypes.byref(arguments(n=0)), None) == _lib.SLK_OK


def test_sizes_grow_with_what_they_hold():
    lib = _lib.load()

    def saved(**kw):
        return lib.slk_attention_saved_bytes(ctypes.byref(arguments(**kw)))

    # two parts of 2 bytes an element, 128 rows for 100
    assert saved() >= 2 * 128 * 64 * 4 * (4 + 2 + 2) + 2 * 128 * 4 * 4
    # one part, and what rounding took off the output: 2 bytes each
    assert saved(dtype=1) >= 2 * 128 * 64 * 2 * (4 + 2 + 2 + 4) + 2 * 128 * 4 * 4
    assert saved(dtype=1) < 0.8 * saved()
    assert saved(keep=0) == 0
    few = arguments(keep=0, rows_q=1, rows_k=1 << 16)
    assert 0 < lib.slk_attention_scratch_bytes(ctypes.byref(few), 0) < 1 << 22
    assert lib.slk_attention_scratch_bytes(None, 0) == 0
    assert lib.slk_attention_saved_bytes(None) == 0


def test_activation_checks_on_the_host():
    lib = _lib.load()

    def no(*words, f=lib.slk_activation_forward, **kw):
        a = dict(n=4, x=16, y=16, dy=16, dx=16, codes=16, scales=16, dtype=0, kind=1)
        refused(f(ctypes.byref(_lib.Activation(**{**a, **kw})), None), *words)

    back = lib.slk_activation_backward
    refused(back(None, None), "NULL arguments")
    no("negative", n=-1)
    no("dtype", dtype=9)
    no("kind", kind=5)
    no("kind", kind=-1)
    no("too large", n=1 << 40)
    no("go together", scales=None)
    no("NULL pointer", x=None)
    no("NULL pointer", y=None, codes=None, scales=None)
    no("NULL pointer", f=back, dx=None)
    no("NULL pointer", f=back, x=None, codes=None, scales=None)
    assert back(ctypes.byref(_lib.Activation(n=0)), None) == _lib.SLK_OK


@pytest.mark.parametrize("buckets,md", [(2, 2), (3, 5), (8, 20), (16, 128), (32, 128), (64, 256),
                                        (128, 256), (16, 9)])
def test_buckets(buckets, md):
    """Every distance in the bucket that the logarithms give, in float64 away from borders and
    exactly on them (where (n / e)^r is a whole power)."""
    starts = relative_buckets(buckets, md)
    e, r = buckets // 2, buckets - buckets // 2
    assert len(starts) == buckets and starts[0] == 0 and starts[-1] <= md
    for n in range(md + 50):
        got = sum(s <= n for s in starts) - 1
        if n < e:
            want = n
        else:
            x = math.log(n / e) / math.log(md / e) * r
            on = round(x)
            if abs(x - on) < 1e-6:  # decided in whole numbers
                x = on if n ** r * e ** on >= e ** r * md ** on else on - 0.5
            want = min(buckets - 1, e + math.floor(x))
        assert got == want, n
    for bad in ((1, 10), (8, 4), (8, 3)):
        with pytest.raises(ValueError):
            relative_buckets(*bad)


def test_layouts_of_gradients():
    for shape, stride in (((2, 3, 4, 8), (3, 1, 48, 6)), ((5, 1, 8), (1, 40, 5)),
                          ((5, 2, 8), (48, 8, 1)), ((2, 3, 4, 8), (0, 8, 0, 1))):
        t = torch.empty_strided(shape, _compact(shape, stride))
        assert _dense(t)
        order = [i for _, i in sorted((s, i) for i, s in enumerate(stride) if s and shape[i] > 1)]
        assert order == sorted(order, key=lambda i: t.stride(i))
    assert not _dense(torch.empty(4, 6)[:, ::2]) and _dense(torch.empty(4, 6).t())
