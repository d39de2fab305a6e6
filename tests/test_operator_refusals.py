"""The operators of the training step on the host: tensors off the GPU are refused, and
the C-ABI's argument checks answer before any device work (fake, never dereferenced
pointers)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import sparsecore_amd as slk
from sparsecore_amd import _lib, optim


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="HIP"):
        slk.residual_norm(x, w)
    with pytest.raises(RuntimeError, match="HIP"):
        slk.linear_cross_entropy(x, torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="HIP"):
        optim.adamw_step([x], [x], [x], [x], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="HIP"):
        optim.quantize(x, True)
    with pytest.raises(RuntimeError, match="HIP"):
        optim.dequantize(x.to(torch.int8), w)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP"):
        optim.carry_slots(i, (i, i), (i, i), [w])


def test_optimizer_arguments():
    p = [torch.nn.Parameter(torch.zeros(4))]
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0),
                dict(state_bits=4), dict(lr=torch.ones(1))):
        with pytest.raises(ValueError):
            slk.AdamW(p, **bad)
    opt = slk.AdamW([{"params": p, "state_bits": 8, "lr": 0.5}])
    assert opt.param_groups[0]["state_bits"] == 8 and opt.param_groups[0]["lr"] == 0.5
    p[0].grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="HIP"):
        opt.step()


def _error(rc, *words):
    lib = _lib.load()
    msg = lib.slk_last_error().decode()
    assert rc == _lib.SLK_EINVAL and all(w in msg for w in words), msg


def test_adamw_checks_on_the_host():
    lib = _lib.load()
    args = _lib.AdamArgs(1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None)
    one = (_lib.AdamTensor * 1)(_lib.AdamTensor(16, 16, 16, 16, None, None, 5))

    def call(dtype=0, bits=32, a=args, t=one, n=1):
        return lib.slk_adamw(ctypes.addressof(t) if t is not None else None, n, dtype, bits,
                             ctypes.byref(a), None)

    _error(call(dtype=7), "dtype")
    _error(call(bits=16), "state_bits")
    _error(call(bits=8), "NULL pointer in tensor 0")  # no scales
    _error(call(t=None), "NULL table")
    _error(call(n=-1), "negative")
    _error(call(a=_lib.AdamArgs(1e-3, 1.0, 0.99, 1e-8, 0.0, 1.0, None, None)), "betas")
    _error(call(a=_lib.AdamArgs(1e-3, 0.9, 0.99, 1e-8, 0.0, 0.0, None, None)), "step")
    _error(call(t=(_lib.AdamTensor * 1)(_lib.AdamTensor(16, 16, 16, 16, None, None, -5))),
           "negative size")
    assert call(n=0) == _lib.SLK_OK


def test_q8_and_carry_checks_on_the_host():
    lib = _lib.load()
    _error(lib.slk_q8_decode(None, None, 4, 1, None, None), "NULL")
    _error(lib.slk_q8_encode(None, -1, 1, None, None, None), "negative")
    state = (_lib.CarryState * 1)(_lib.CarryState(16, None, 16, None, 0))
    _error(lib.slk_carry_slots(16, 2, 10, 16, 16, 16, 16, state, 1, None), "in place")
    state[0].dst, state[0].kind = 32, _lib.STATE_Q8_SIGNED
    _error(lib.slk_carry_slots(16, 2, 10, 16, 16, 16, 16, state, 1, None), "NULL pointer in state")
    state[0].kind = 9
    _error(lib.slk_carry_slots(16, 2, 10, 16, 16, 16, 16, state, 1, None), "kind")
    _error(lib.slk_carry_slots(16, 2, 10, 16, 16, 16, 16, state, 9, None), "states")
    _error(lib.slk_carry_slots(16, 0, 10, 16, 16, 16, 16, state, 1, None), "without rows")
    _error(lib.slk_carry_slots(16, 2, 1 << 31, 16, 16, 16, 16, state, 1, None), "int32")
    _error(lib.slk_carry_slots(None, 2, 10, 16, 16, 16, 16,
                               (_lib.CarryState * 1)(_lib.CarryState(16, None, 32, None, 0)), 1,
                               None), "NULL structure")
    assert lib.slk_carry_slots(None, 0, 0, None, None, None, None, state, 1, None) == _lib.SLK_OK


def test_norm_checks_on_the_host():
    lib = _lib.load()

    def call(f=lib.slk_norm_forward, **kw):
        a = dict(n=4, d=8, x=16, weight=16, r=16, y=16, dtype=0, layer=1, scale=1.0, eps=1e-5)
        return f(ctypes.byref(_lib.Norm(**{**a, **kw})), None)

    _error(call(d=0), "d in [1")
    _error(call(d=_lib.NORM_MAX_D + 1), "d in [1")
    _error(call(dtype=5), "dtype")
    _error(call(weight=None), "NULL weight")
    _error(call(x=None), "NULL x")
    _error(call(gate=16), "gate needs a branch")
    _error(call(post_weight=16), "post norm needs a branch")
    _error(call(branch=16, post_bias=16), "post_bias needs")
    _error(call(layer=0, bias=16), "no bias")
    _error(call(branch=16, gate=16, gate_rows=3), "must divide")
    _error(call(d=_lib.NORM_COLS_MAX + 1, y_cols=1), "feature-major")
    back = lib.slk_norm_backward
    _error(call(back), "stats")
    _error(call(back, stats=16, dbranch=16), "without a branch")
    _error(call(back, stats=16, dy=16, dweight=16), "workspace too small")
    assert call(n=0, x=None) == _lib.SLK_OK


def test_linear_ce_checks_on_the_host():
    lib = _lib.load()

    def call(f=lib.slk_linear_ce_forward, **kw):
        a = dict(n=4, d=8, v=10, hidden=16, weight=16, target=16, loss=16, dtype=0, reduction=0,
                 keep=0)
        return f(ctypes.byref(_lib.LinearCE(**{**a, **kw})), None)

    _error(call(d=0), "d and v")
    _error(call(v=1 << 26), "2^25")
    _error(call(dtype=3), "dtype")
    _error(call(reduction=4), "reduction")
    _error(call(hidden=None), "NULL hidden")
    _error(call(), "scratch too small")
    back = lib.slk_linear_ce_backward
    _error(call(back), "kept nothing")
    _error(call(back, keep=1), "upstream")
    _error(call(back, keep=1, upstream=16), "too small")
    assert call(n=0, hidden=None) == _lib.SLK_OK


def test_workspace_sizes_are_bounded():
    """The backward's scratch holds a piece of the vocabulary's logit gradients, not all:
    far below 4 bytes a logit for a large vocabulary, and never below what it names."""
    a = _lib.LinearCE(n=8192, d=512, v=400000, dtype=0, reduction=2, keep=1, dhidden=16,
                      dweight=16)
    scratch = _lib.linear_ce_scratch_bytes(a, True)
    assert (1 << 28) < scratch < (1 << 30) + 16 * 8192 * 512 * 4
    assert scratch < 8192 * 400000
    few = _lib.LinearCE(n=16, d=512, v=400000, dtype=0, reduction=0, keep=0)
    assert _lib.linear_ce_saved_bytes(few) == 0
    assert _lib.linear_ce_scratch_bytes(few, False) < 1 << 20
