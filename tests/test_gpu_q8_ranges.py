"""8-bit codes of blocks at the ends of float32's range, against the maps in numpy."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from sparsecore_amd import optim
from test_gpu_adamw import np_decode, np_encode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("top", [2.0 ** -126, 2.0 ** -100, 2.0 ** 100, 2.0 ** 124, 2.0 ** 125,
                                 2.0 ** 126, 1.5 * 2.0 ** 126, 2.0 ** 127, 3.4e38])
def test_codes_of_any_scale(dev, signed, top):
    rng = np.random.default_rng(3)
    x = (rng.random(1024) ** 2 * rng.choice([-1, 1], 1024)).astype(np.float32)
    x[::256] = 1.0
    x = (x.astype(np.float64) * top).astype(np.float32)
    x[5] = 0.0
    if not signed:
        x = np.abs(x)
    codes, scales = optim.quantize(torch.from_numpy(x).to(dev), signed)
    want, scale = np_encode(x, signed)
    assert np.array_equal(scales.cpu().numpy(), scale)
    normal = np.abs(x) >= 2.0 ** -126  # of a subnormal the instructions take no root
    got = codes.cpu().numpy()
    assert np.array_equal(got[normal], want[normal]) and (got[x == 0] == 0).all()
    assert np.array_equal(optim.dequantize(codes, scales).cpu().numpy()[normal],
                          np_decode(want, scale)[normal])
