"""AdamW's bookkeeping on the host: which count each parameter is stepped with. The launch
and the checks of device tensors are replaced by a recorder, so these run on CPU tensors."""

from __future__ import annotations

import copy
import pickle

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


@pytest.fixture
def layer(launches, monkeypatch):
    """A SparseLinear, and a carry of its moments that runs on the host."""
    def carry(row_start, old, new, states):
        out = []
        for s in states:
            to = torch.zeros_like(s)
            for r, start in enumerate(row_start.tolist()):
                was = {int(old[0][k]): k for k in range(start, start + int(old[1][r]))}
                for k in range(start, start + int(new[1][r])):
                    if int(new[0][k]) in was:
                        to[k] = s[was[int(new[0][k])]]
            out.append(to)
        return out

    monkeypatch.setattr(optim, "carry_slots", carry)
    torch.manual_seed(0)
    net = slk.SparseLinear(20, 12, sparsity=0.5, bias=False)
    net._values.grad = torch.ones_like(net._values)
    return net


def rewrite(net):
    """Moves the first connection of every row to a column that the row did not have."""
    csr = net._csr
    for r, start in enumerate(csr.row_start.tolist()):
        n = int(csr.row_nnz[r])
        cols = csr.col_indices[start:start + n]
        free = next(c for c in range(csr.ncols) if c not in cols.tolist())
        cols[0] = free
        cols.copy_(cols.sort().values)
    csr._topology_version += 1


@pytest.mark.parametrize("how", ["step", "follow"])
def test_carried_moments_stay_where_they_are(layer, how):
    """A captured step's replays read the addresses of its capture."""
    p = layer._values
    opt = slk.AdamW([p], capturable=True)
    opt.attach(layer)
    opt.step()
    s = opt.state[p]
    s["exp_avg"].copy_(torch.arange(float(p.numel())))
    before, at = dict(s), s["exp_avg"].data_ptr()
    old = layer._csr.col_indices.clone(), layer._csr.row_nnz.clone()
    want, = optim.carry_slots(layer._csr.row_start, old, old, [s["exp_avg"].clone()])
    rewrite(layer)
    want, = optim.carry_slots(layer._csr.row_start, old,
                              (layer._csr.col_indices, layer._csr.row_nnz), [s["exp_avg"].clone()])
    getattr(opt, how)()
    assert all(s[k] is before[k] for k in before) and s["exp_avg"].data_ptr() == at
    assert torch.equal(s["exp_avg"], want) and bool((want == 0).any())
    opt.follow()  # nothing is left to move
    assert torch.equal(s["exp_avg"], want)


def test_a_capture_that_would_record_a_move_or_a_beginning_is_refused(layer, monkeypatch):
    p = layer._values
    opt = slk.AdamW([p], capturable=True)
    opt.attach(layer)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    capturing = [True]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    with pytest.raises(RuntimeError, match="before capturing"):
        opt.step()  # would zero the moments and the count on every replay
    assert not opt.state[p]
    capturing[0] = False
    opt.step()
    rewrite(layer)
    capturing[0] = True
    with pytest.raises(RuntimeError, match="follow"):
        opt.step()  # would move the moments on every replay
    with pytest.raises(RuntimeError, match="follow"):
        opt.follow()
    capturing[0] = False
    opt.follow()
    capturing[0] = True
    opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_what_a_step_writes_changes_its_version(monkeypatch, bits):
    """As torch's in-place operations do, so that a backward which saved a parameter
    raises after a step in place of computing with the new one."""
    from sparsecore_amd import _lib

    monkeypatch.setattr(_lib, "adamw", lambda *a: None)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(_lib, "on_device", lambda t: _lib._SAME_DEVICE)
    p, g = torch.nn.Parameter(torch.zeros(300)), torch.zeros(300)
    kinds = (torch.int8, torch.uint8) if bits == 8 else (torch.float32,) * 2
    m, v = (torch.zeros(300, dtype=k) for k in kinds)
    scales = (torch.zeros(2), torch.zeros(2)) if bits == 8 else ()
    optim._launch([300], [p], [g], [m], [v], tuple([s] for s in scales) or None, 1, 1e-3,
                  (0.9, 0.99), 1e-8, 0.0)
    assert all(t._version == 1 for t in (p, m, v, *scales)) and g._version == 0


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_copies_of_an_optimizer_step(layer, launches, how):
    opt = slk.AdamW([layer._values])
    opt.attach(layer)
    opt.step()
    twin = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
    p, = twin.param_groups[0]["params"]
    p.grad = torch.ones_like(p)
    launches.clear()
    twin.step()
    assert counts(launches, [p, layer._values]) == [[2], []]
    twin.load_state_dict(opt.state_dict())
    twin.step()
    assert twin.state[p]["step"] == 2 and opt.state[layer._values]["step"] == 1
    twin.attach(layer)  # a copy's own layers are attached anew
    assert layer._values in twin._attached


def test_attaching_again_keeps_a_move_that_is_due(layer):
    p = layer._values
    opt = slk.AdamW([p])
    opt.attach(layer)
    opt.step()
    s = opt.state[p]
    s["exp_avg"].copy_(torch.arange(float(p.numel())))
    old = layer._csr.col_indices.clone(), layer._csr.row_nnz.clone()
    rewrite(layer)
    want, = optim.carry_slots(layer._csr.row_start, old,
                              (layer._csr.col_indices, layer._csr.row_nnz), [s["exp_avg"].clone()])
    opt.attach(layer)
    opt.step()
    assert torch.equal(s["exp_avg"], want)


@pytest.mark.parametrize("how", ["state_dict", "deepcopy", "pickle"])
def test_what_is_saved_after_a_rewrite_fits_the_new_slots(layer, how):
    """A loop that steps, rewrites and then saves: the model is saved with the topology
    after the rewrite, so the moments must be at that topology's slots."""
    p = layer._values
    opt = slk.AdamW([p])
    opt.attach(layer)
    opt.step()
    s = opt.state[p]
    s["exp_avg"].copy_(torch.arange(float(p.numel())))
    old = layer._csr.col_indices.clone(), layer._csr.row_nnz.clone()
    rewrite(layer)
    want, = optim.carry_slots(layer._csr.row_start, old,
                              (layer._csr.col_indices, layer._csr.row_nnz), [s["exp_avg"].clone()])
    if how == "state_dict":
        got = opt.state_dict()["state"][0]["exp_avg"]
    else:
        twin = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
        got = twin.state[twin.param_groups[0]["params"][0]]["exp_avg"]
    assert torch.equal(got, want) and torch.equal(s["exp_avg"], want)


def test_a_replaced_matrix_does_not_stop_a_checkpoint(layer):
    opt = slk.AdamW([layer._values])
    opt.attach(layer)
    opt.step()
    layer.load_state_dict({k: v.clone() for k, v in layer.state_dict().items()})
    saved = opt.state_dict()
    with pytest.raises(RuntimeError, match="attach"):
        opt.step()
    opt.load_state_dict(saved)
    opt.step()
    assert opt.state[layer._values]["step"] == 2
