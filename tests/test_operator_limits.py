"""Sizes beyond what a launch takes are refused on the host, before any device work (fake,
never dereferenced pointers): a launch has at most 2^32 - 1 threads along its grid."""

from __future__ import annotations

import ctypes

import pytest

from sparsecore_amd import _lib


def refused(rc, *words):
    msg = _lib.load().slk_last_error().decode()
    assert rc == _lib.SLK_EINVAL and all(w in msg for w in words), msg


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw(bits):
    args = _lib.AdamArgs(1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None)
    n = 4 * (2 ** 32 - 1) + 1024  # four elements a thread
    one = (_lib.AdamTensor * 1)(_lib.AdamTensor(16, 16, 16, 16, 16, 16, n))
    refused(_lib.load().slk_adamw(ctypes.addressof(one), 1, 0, bits, ctypes.byref(args), None),
            "tensor 0 is too large")


def test_codes():
    lib, n = _lib.load(), 4 * (2 ** 32 - 1) + 1024
    refused(lib.slk_q8_decode(16, 16, n, 1, 16, None), "too large")
    refused(lib.slk_q8_encode(16, n, 1, 16, 16, None), "too large")


@pytest.mark.parametrize("d,cols,threads", [(4, 0, 64), (4, 1, 32), (768, 0, 64), (768, 1, 32),
                                            (2048, 0, 256), (4096, 0, 512), (16384, 0, 1024)])
def test_norm(d, cols, threads):
    a = _lib.Norm(n=(2 ** 32 - 1) // threads + 1, d=d, x=16, weight=16, r=16, y=16, stats=16,
                  dtype=1, layer=0, scale=1.0, eps=1e-5, y_cols=cols)
    lib = _lib.load()
    refused(lib.slk_norm_forward(ctypes.byref(a), None), "at most", "tokens")
    refused(lib.slk_norm_backward(ctypes.byref(a), None), "at most", "tokens")


def test_head():
    a = _lib.LinearCE(n=1 << 20, d=64, v=1 << 19, hidden=16, weight=16, target=16, loss=16,
                      dtype=1, reduction=2, keep=1, upstream=16)
    lib = _lib.load()  # 2^23 tiles of 256 x 256, 512 threads each
    refused(lib.slk_linear_ce_forward(ctypes.byref(a), None), "too many logits")
    refused(lib.slk_linear_ce_backward(ctypes.byref(a), None), "too many logits")
    a.v -= 256
    refused(lib.slk_linear_ce_forward(ctypes.byref(a), None), "scratch too small")


def test_alignment():
    """The arrays that the kernels themselves lay out are read sixteen bytes at a time."""
    lib = _lib.load()
    a = _lib.LinearCE(n=200, d=64, v=300, hidden=16, weight=16, target=16, loss=16, upstream=16,
                      dtype=0, reduction=0, keep=1, saved_bytes=1 << 40, scratch_bytes=1 << 40)
    for a.saved, a.scratch in ((24, 32), (32, 24)):
        refused(lib.slk_linear_ce_forward(ctypes.byref(a), None), "aligned")
        refused(lib.slk_linear_ce_backward(ctypes.byref(a), None), "aligned")
    b = _lib.Norm(n=4, d=8, x=16, weight=16, r=16, y=16, stats=20, dtype=0, layer=1, scale=1.0,
                  eps=1e-5)
    refused(lib.slk_norm_forward(ctypes.byref(b), None), "aligned")
    refused(lib.slk_norm_backward(ctypes.byref(b), None), "aligned")
