"""What linear_cross_entropy keeps and takes, by the sizes alone (host)."""

from __future__ import annotations

import pytest

from sparsecore_amd import _lib


def sizes(n, d, v, dtype, keep=1):
    a = _lib.LinearCE(n=n, d=d, v=v, dtype=dtype, reduction=2, keep=keep, dhidden=16, dweight=16)
    return _lib.linear_ce_saved_bytes(a), _lib.linear_ce_scratch_bytes(a, True)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n", [200, 8192, 100000, 1 << 19, 1 << 20, 1 << 22, 1 << 25])
@pytest.mark.parametrize("d,v", [(64, 32000), (768, 400000)])
def test_the_backwards_scratch(n, d, v, dtype):
    """A piece of the vocabulary's logit gradients (one array in bfloat16, two in float32)
    of at most 2^29 bytes each, or of 256 rows over all tokens where those take more; the
    float32 sums of dh, and of a piece's dw where its sum has parts; some exponents."""
    arrays, each = (1, 2) if dtype else (2, 4)
    tokens = -(-n // 256) * 256
    dl = arrays * max(1 << 29, 256 * tokens * each)
    rows = max(1 << 29, 256 * tokens * each) // (tokens * each)
    sums = 4 * d * 32 * (n + min(rows, v + 255))
    exps = 4 * (tokens * (rows // 256 + 2) + rows * (tokens // 128 + 2)) + 4096
    assert sizes(n, d, v, dtype)[1] <= dl + sums + exps


@pytest.mark.parametrize("dtype", [0, 1])
def test_what_a_forward_keeps(dtype):
    size = 2 if dtype else 4
    few = sizes(32, 512, 400000, dtype)[0]  # the logits: 32 a row of the head
    assert 32 * 4 * 400000 <= few <= 32 * 4 * 400000 + 4096
    small = sizes(10000, 64, 65, dtype)[0]  # 80 a token
    assert 80 * 4 * 10000 <= small <= 88 * 4 * 10000 + 4096
    packed = sizes(4096, 512, 32000, dtype)[0]  # both operands once more
    assert packed <= (4096 + 32000) * (512 * size + 4) + 4096 * 24 + 65536
