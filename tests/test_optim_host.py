"""AdamW's bookkeeping on the host: which count each parameter is stepped with. The launch
and the checks of device tensors are replaced by a recorder, so these run on CPU tensors."""

from __future__ import annotations

import copy

import pytest
import torch

import sparsecore_amd as slk
from sparsecore_amd import optim


@pytest.fixture
def launches(monkeypatch):
    """[(parameters, count)] of every launch."""
    seen = []

    def launch(sizes, params, grads, m, v, scales, step, *rest):
        seen.append((list(params), float(step)))

    monkeypatch.setattr(optim, "_check_lists", lambda params, *rest: [p.numel() for p in params])
    monkeypatch.setattr(optim, "_launch", launch)
    return seen


def parameters(n):
    out = [torch.nn.Parameter(torch.zeros(4)) for _ in range(n)]
    for p in out:
        p.grad = torch.ones(4)
    return out


def counts(launches, params):
    """The counts that each parameter was stepped with, in order."""
    return [[c for ps, c in launches if any(p is q for q in ps)] for p in params]


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("through", ["memory", "copied tensors"])
def test_groups_count_their_own_steps_after_loading(launches, capturable, through):
    p = parameters(3)

    def make():
        return slk.AdamW([{"params": p[:2]}, {"params": p[2:], "weight_decay": 0.0}],
                         capturable=capturable)

    opt = make()
    for _ in range(3):
        opt.step()
    saved = opt.state_dict()
    if through != "memory":  # as files that hold tensors by name give them back
        saved = {"param_groups": saved["param_groups"],
                 "state": {i: {k: copy.deepcopy(v) for k, v in s.items()}
                           for i, s in saved["state"].items()}}
    twin = make()
    twin.load_state_dict(saved)
    launches.clear()
    for _ in range(3):
        twin.step()
    assert counts(launches, p) == [[4.0, 5.0, 6.0]] * 3
    assert len(launches) == 6  # a launch a group: parameters of one count stay together
    assert [float(opt.state[q]["step"]) for q in p] == [3.0] * 3  # nothing shared with the source


@pytest.mark.parametrize("capturable", [False, True])
def test_a_parameter_without_a_gradient_keeps_its_count(launches, capturable):
    p = parameters(3)
    opt = slk.AdamW(p, capturable=capturable)
    opt.step()
    p[1].grad = None
    opt.step()
    opt.step()
    p[1].grad = torch.ones(4)
    opt.step()
    assert counts(launches, p) == [[1, 2, 3, 4], [1, 2], [1, 2, 3, 4]]


def test_a_capture_that_would_part_counts_is_refused(launches, monkeypatch):
    p = parameters(2)
    opt = slk.AdamW(p, capturable=True)
    opt.step()
    p[1].grad = None
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        opt.step()
    with monkeypatch.context() as eager:
        eager.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        opt.step()
    opt.step()  # the counts are apart now
    assert counts(launches, p) == [[1, 2, 3], [1]]
