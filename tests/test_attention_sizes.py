"""slk_attention_*_bytes and the entry points on the host, for sizes that no call may have:
0 bytes and a refusal, without a division by zero or a product past 64 bits."""

from __future__ import annotations

import ctypes

import pytest

from sparsecore_amd import _lib

BIG = (1 << 63) - 1


def arguments(**kw):
    a = dict(n=2, rows_q=100, rows_k=100, heads=4, kv_heads=2, dim=64, scale=0.125, dtype=0,
             causal=1, keep=1, saved=16, saved_bytes=1 << 50, scratch=16, scratch_bytes=1 << 50)
    for k in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        a[k] = _lib.AttnTensor(16, 0, 64, 64, 1)
    return _lib.Attention(**{**a, **kw})


@pytest.mark.parametrize("wrong", [
    {"kv_heads": 0}, {"kv_heads": -2}, {"heads": 0}, {"heads": 3}, {"heads": 1 << 40},
    {"n": BIG}, {"n": 1 << 40}, {"n": -1}, {"rows_q": BIG}, {"rows_q": 1 << 40, "n": 1 << 30},
    {"rows_k": BIG}, {"rows_k": -1}, {"dim": 0}, {"dim": BIG},
    {"n": 1 << 24, "rows_q": 1 << 24}, {"n": BIG, "q_offsets": 16},
    {"rows_q": BIG, "rows_k": BIG, "q_offsets": 16},
    {"bias": 16, "buckets": 8, "max_distance": BIG}, {"bias": 16, "max_distance": 0}])
@pytest.mark.parametrize("keep", [0, 1])
def test_sizes_that_are_refused(wrong, keep):
    lib = _lib.load()
    a = arguments(keep=keep, **wrong)
    assert lib.slk_attention_saved_bytes(ctypes.byref(a)) == 0
    for backward in (0, 1):
        assert lib.slk_attention_scratch_bytes(ctypes.byref(a), backward) == 0
    for f in (lib.slk_attention_forward, lib.slk_attention_backward):
        assert f(ctypes.byref(a), None) == _lib.SLK_EINVAL


def test_largest_sizes_are_counted():
    lib = _lib.load()
    a = arguments(n=1, rows_q=1 << 29, rows_k=1 << 29, heads=16384, kv_heads=1, dim=128)
    # two parts of 2 bytes an element
    assert lib.slk_attention_saved_bytes(ctypes.byref(a)) >= 4 * 128 * (16384 + 2) << 29
    assert lib.slk_attention_scratch_bytes(ctypes.byref(a), 1) >= 4 * 128 * 16384 << 29


def test_scales_that_leave_float32_are_refused():
    lib = _lib.load()
    for scale in (3e38, 2.1e38, 1e300):
        a = arguments(scale=scale)
        assert lib.slk_attention_forward(ctypes.byref(a), None) == _lib.SLK_EINVAL
        assert b"scale" in lib.slk_last_error()
