"""sparsecore_amd.optim — AdamW over many tensors at once, moments in 32 or 8 bits,
and moments that follow their weights through SET / RigL rewrites.

    AdamW            torch.optim.Optimizer; model.apply(opt.attach) makes the moments of
                     every SparseLinear follow its topology
    adamw_step       the step itself on lists of tensors
    carry_slots      per-slot states of a padded-CSR matrix moved to its new topology
    quantize, dequantize   8-bit moments and the float32 values they stand for

One step of a whole model is one kernel launch per 56 tensors of a dtype
(``slk_adamw``), with no copy of a pointer table to the device.

8-bit moments: blocks of 256 elements share a float32 scale, the block's largest
magnitude; the first moment's int8 code q stands for (q/127)·|q/127|·scale, the
second's uint8 code for (q/255)⁴·scale. A step takes 16 bytes of traffic per float32
parameter instead of 28, and 2 bytes of state instead of 8. An attached SparseLinear adds
a copy of its column indices, 4 bytes a slot, with either.
"""

from __future__ import annotations

import numpy as np
import torch

from . import _lib

__all__ = ["AdamW", "adamw_step", "carry_slots", "quantize", "dequantize"]

BLOCK = _lib.Q8_BLOCK


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _on_device(who: str, name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{who}: {name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{who}: {name} must be on a HIP (ROCm) device (got "
                           f"device={t.device})")


# ─────────────────────────── 8-bit moments ───────────────────────────

def _check_q8(who: str, codes: torch.Tensor, scales: torch.Tensor) -> None:
    _on_device(who, "codes", codes)
    _on_device(who, "scales", scales)
    if codes.dtype not in (torch.int8, torch.uint8):
        raise ValueError(f"{who}: codes must be int8 (first moment) or uint8 (second moment), "
                         f"got {codes.dtype}")
    if scales.dtype != torch.float32 or scales.numel() != _blocks(codes.numel()):
        raise ValueError(f"{who}: {codes.numel()} codes need {_blocks(codes.numel())} float32 "
                         f"scales, got {scales.numel()} of {scales.dtype}")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{who}: codes and scales must be contiguous")
    if codes.device != scales.device:
        raise RuntimeError(f"{who}: codes are on {codes.device} but scales on {scales.device}")


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float32 values that 8-bit moments stand for, in the shape of codes: int8
    codes are a first moment's, uint8 codes a second moment's."""
    _check_q8("dequantize", codes, scales)
    out = torch.empty(codes.shape, dtype=torch.float32, device=codes.device)
    with _lib.on_device(codes):
        _lib.q8_decode(codes, scales, out)
    return out


def quantize(x: torch.Tensor, signed: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of a float32 tensor: int8 codes of the first moment's map
    (``signed``), else uint8 codes of the second's, for x >= 0."""
    _on_device("quantize", "x", x)
    if x.dtype != torch.float32:
        raise ValueError(f"quantize: x must be float32, got {x.dtype}")
    x = x.contiguous()
    codes = torch.empty(x.shape, dtype=torch.int8 if signed else torch.uint8, device=x.device)
    scales = torch.empty(_blocks(x.numel()), dtype=torch.float32, device=x.device)
    with _lib.on_device(x):
        _lib.q8_encode(x, codes, scales)
    return codes, scales


# ─────────────────────────── the step ───────────────────────────

def _scalar(name: str, v, dev: int):
    """(host value, device address): one of the two carries the scalar."""
    if not isinstance(v, torch.Tensor):
        return float(v), None
    if v.numel() != 1 or v.dtype != torch.float32 or not v.is_cuda or v.get_device() != dev:
        raise ValueError(f"adamw_step: a tensor {name} must be one float32 value on the "
                         f"parameters' device")
    return 1.0, v.data_ptr()


def _check_hyper(lr, betas, eps, weight_decay, step) -> None:
    if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
        raise ValueError(f"adamw_step: lr must be >= 0, got {lr}")
    if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
        raise ValueError(f"adamw_step: betas must be two values in [0, 1), got {betas}")
    if not eps >= 0.0:
        raise ValueError(f"adamw_step: eps must be >= 0, got {eps}")
    if not weight_decay >= 0.0:
        raise ValueError(f"adamw_step: weight_decay must be >= 0, got {weight_decay}")
    if not isinstance(step, torch.Tensor) and not step >= 1:
        raise ValueError(f"adamw_step: step must be >= 1, got {step}")


def _check_lists(params, grads, moments, scales) -> list:
    """Everything the kernel relies on, over whole lists at a time (a step of a small
    model is bound by this host work). Returns the parameters' sizes."""
    n = len(params)
    lists = [params, grads, *moments, *(scales or ())]
    if {len(t) for t in lists} - {n}:
        raise ValueError("adamw_step: params, grads, moments (and scales) must be lists of the "
                         "same length")
    every = [t for part in lists for t in part]
    try:
        devices = {t.get_device() for t in every}
        packed = all([t.is_contiguous() for t in every])
        sizes = [t.numel() for t in params]
        kinds = [t.dtype for t in params]
    except (AttributeError, TypeError):
        raise TypeError("adamw_step: lists of torch.Tensor expected") from None
    if -1 in devices:
        raise RuntimeError("adamw_step: every tensor must be on a HIP (ROCm) device")
    if len(devices) > 1:
        raise RuntimeError("adamw_step: all tensors of a call must be on one device")
    if not packed:
        raise ValueError("adamw_step: tensors must be contiguous")
    for what, have in (("grads", grads), ("exp_avgs", moments[0]), ("exp_avg_sqs", moments[1])):
        if [t.numel() for t in have] != sizes:
            raise ValueError(f"adamw_step: {what} must have their parameters' sizes")
    if [t.dtype for t in grads] != kinds:
        raise ValueError("adamw_step: a gradient must have its parameter's dtype")
    bad = set(kinds) - set(_lib.DTYPES)
    if bad:
        raise ValueError(f"adamw_step: parameters must be float32 or bfloat16, got {bad.pop()}")
    want = ({torch.int8}, {torch.uint8}) if scales else ({torch.float32}, {torch.float32})
    if n and ({t.dtype for t in moments[0]}, {t.dtype for t in moments[1]}) != want:
        raise ValueError("adamw_step: moments must be float32, or int8 (exp_avgs) and uint8 "
                         "(exp_avg_sqs) with their scales")
    if scales:
        for t in scales:
            if {x.dtype for x in t} - {torch.float32}:
                raise ValueError("adamw_step: scales must be float32")
            if [x.numel() for x in t] != [_blocks(k) for k in sizes]:
                raise ValueError(f"adamw_step: one scale per {BLOCK} elements expected")
    return sizes


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, exp_avg_scales=None,
               exp_avg_sq_scales=None, step, lr, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.01) -> None:
    """One AdamW step of a list of tensors, in place:

        m = β1·m + (1 - β1)·g,   v = β2·v + (1 - β2)·g²
        p = (1 - lr·wd)·p - lr / (1 - β1^t) · m / (√v / √(1 - β2^t) + eps)

    Parameters and gradients are float32 or bfloat16 (arithmetic in float32, a
    bfloat16 parameter rounded once). Moments are float32, or 8-bit codes with their
    scales (``quantize``); the update uses the unrounded moments. ``step`` counts from 1.
    ``step`` and ``lr`` may be one-element float32 tensors on the device, which a
    captured graph reads at each replay. The padding slots of a padded-CSR matrix's
    values have gradient 0 and stay 0.

    Raises TypeError (not tensors), RuntimeError (not on one HIP device) and ValueError
    (sizes, dtypes, layouts, hyperparameters).
    """
    if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
        raise ValueError("adamw_step: scales of both moments or of none")
    scales = None if exp_avg_scales is None else (exp_avg_scales, exp_avg_sq_scales)
    _check_hyper(lr, betas, eps, weight_decay, step)
    sizes = _check_lists(params, grads, (exp_avgs, exp_avg_sqs), scales)
    _launch(sizes, params, grads, exp_avgs, exp_avg_sqs, scales, step, lr, betas, eps,
            weight_decay)


def _launch(sizes, params, grads, exp_avgs, exp_avg_sqs, scales, step, lr, betas, eps,
            weight_decay):
    if not params:
        return
    dev = params[0].get_device()
    step, step_dev = _scalar("step", step, dev)
    lr, lr_dev = _scalar("lr", lr, dev)
    args = _lib.AdamArgs(lr, betas[0], betas[1], eps, weight_decay, step, step_dev, lr_dev)
    cols = [params, grads, exp_avgs, exp_avg_sqs, *(scales or ())]
    rows = [[t.data_ptr() for t in tensors] for tensors in cols]
    if not scales:
        rows += [[0] * len(params)] * 2
    table = np.array([*rows, sizes], dtype=np.int64).T.copy()  # a row a tensor
    bits = 8 if scales else 32
    kinds = [t.dtype for t in params]
    with _lib.on_device(params[0]):
        stream = _lib.stream_of(params[0])
        for dtype in dict.fromkeys(kinds):
            part = table
            if any(k is not dtype for k in kinds):
                part = table[[k is dtype for k in kinds]]
            _lib.adamw(part, len(part), _lib.DTYPES[dtype], bits, args, stream)
    # written through their addresses: a backward that has saved one of them must notice
    torch.autograd.graph.increment_version([t for k, ts in enumerate(cols) if k != 1 for t in ts])


# ─────────────────────── states that follow a rewrite ───────────────────────

def carry_slots(row_start, old, new, states) -> list:
    """Per-slot states of a padded-CSR matrix, moved to its topology after a rewrite.

    ``old`` and ``new`` are (col_indices, row_nnz) before and after; ``row_start`` is
    common to both, as a rewrite keeps each row's place. The slot that holds (row,
    column) now takes the state of the slot that held it before; grown connections and
    padding take 0. ``states``: up to four float32 tensors, or (codes, scales) pairs of
    8-bit moments, one entry per slot. Returns new tensors of the same kinds.
    """
    arrays = [("row_start", row_start), ("old col_indices", old[0]), ("old row_nnz", old[1]),
              ("new col_indices", new[0]), ("new row_nnz", new[1])]
    for name, t in arrays:
        _on_device("carry_slots", name, t)
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"carry_slots: {name} must be a contiguous 1-D int32 tensor")
        if t.device != row_start.device:
            raise RuntimeError(f"carry_slots: {name} is on {t.device} but row_start on "
                               f"{row_start.device}")
    rows, total = row_start.numel(), old[0].numel()
    if new[0].numel() != total or old[1].numel() != rows or new[1].numel() != rows:
        raise ValueError("carry_slots: both topologies must have the same rows and slots")
    if total and not rows:
        raise ValueError("carry_slots: slots without rows")
    if len(states) > _lib.CARRY_STATES:
        raise ValueError(f"carry_slots: at most {_lib.CARRY_STATES} states, got {len(states)}")
    table, out = [], []
    for s in states:
        codes, scales = s if isinstance(s, (tuple, list)) else (s, None)
        if scales is None:
            _on_device("carry_slots", "a state", codes)
            if codes.dtype != torch.float32 or not codes.is_contiguous():
                raise ValueError("carry_slots: a state must be contiguous float32, or (codes, "
                                 "scales) of an 8-bit moment")
        else:
            _check_q8("carry_slots", codes, scales)
        if codes.numel() != total or codes.device != row_start.device:
            raise ValueError(f"carry_slots: a state must have one entry per slot ({total}) on "
                             f"{row_start.device}")
        to = torch.empty_like(codes)
        if scales is None:
            out.append(to)
            table.append((codes, None, to, None, _lib.STATE_F32))
        else:
            kind = _lib.STATE_Q8_SIGNED if codes.dtype == torch.int8 else _lib.STATE_Q8_UNSIGNED
            to_scales = torch.empty_like(scales)
            out.append((to, to_scales))
            table.append((codes, scales, to, to_scales, kind))
    with _lib.on_device(row_start):
        _lib.carry_slots(row_start, old[0], old[1], new[0], new[1], table)
    return out


# ─────────────────────────── the optimizer ───────────────────────────

def _capturing() -> bool:
    return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()


class _Attached:
    """A SparseLinear's topology as its moments know it."""

    def __init__(self, layer):
        self.layer = layer
        self.cols = self.nnz = None
        self.snapshot()

    def snapshot(self) -> None:
        csr = self.layer._csr
        self.csr = csr
        self.version = csr.topology_version
        self.cols = _copied(self.cols, csr.col_indices)
        self.nnz = _copied(self.nnz, csr.row_nnz)


def _copied(to, t):
    """t's values, in `to` where they fit it."""
    if to is None or to.shape != t.shape or to.device != t.device:
        return t.clone()
    return to.copy_(t)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay; the whole model in one launch per 56 tensors.

    Args:
        params: parameters (float32 or bfloat16, on one HIP device) or groups of them.
        lr: learning rate, a float or (with ``capturable``) a float32 device tensor.
        betas, eps, weight_decay: as in ``adamw_step``.
        state_bits: 32 (float32 moments) or 8 (codes with a scale per 256 elements).
            A group's choice; small tensors such as norm weights can keep 32.
        capturable: keep the step count on the device, so that a captured graph counts
            its replays. Otherwise a step under capture raises RuntimeError, since the
            graph would repeat one step's bias corrections. Moments begin in an eager
            step: a capture before it raises too.

    A SET or RigL rewrite gives slots to other weights. ``model.apply(opt.attach)``
    makes the moments of each SparseLinear follow: the next ``step()`` first moves them
    to their weights' new slots (``carry_slots``) and starts grown connections at 0.
    Replays of a captured step do not: call ``follow()`` after each rewrite, before the
    next replay. The moments stay in their tensors, so the capture remains valid.
    A layer whose matrix was replaced (``load_state_dict``, ``reset_parameters``) is
    attached again, after loading the optimizer's own state. Moments are saved and copied
    as of the layers' present topology; a deep copy or an unpickled optimizer has no layers
    attached: ``attach`` its own.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, *, state_bits: int = 32, capturable: bool = False):
        _check_hyper(lr, betas, eps, weight_decay, 1)
        self._attached: dict = {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay, state_bits=state_bits,
                                      capturable=capturable))

    def add_param_group(self, group) -> None:
        group = dict(group)
        g = {**self.defaults, **{k: v for k, v in group.items() if k != "params"}}
        _check_hyper(g["lr"], g["betas"], g["eps"], g["weight_decay"], 1)
        if g["state_bits"] not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {g['state_bits']}")
        if isinstance(g["lr"], torch.Tensor) and not g["capturable"]:
            raise ValueError("AdamW: a tensor lr needs capturable=True")
        super().add_param_group(group)

    def _settle(self) -> None:
        """What is saved fits the topology that the model is saved with. (Moments of a
        layer whose matrix was replaced fit none: the next step refuses them.)"""
        with torch.no_grad():
            for p, at in self._attached.items():
                if at.layer._csr is at.csr:
                    self._follow(p)

    def state_dict(self) -> dict:
        self._settle()
        return super().state_dict()

    def __getstate__(self) -> dict:
        self._settle()
        return super().__getstate__()

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        self.__dict__.setdefault("_attached", {})  # a copy: it knows no layers yet

    # ─── topology ───

    def attach(self, module) -> None:
        """Make a SparseLinear's moments follow its topology (other modules are
        ignored, so that ``model.apply(opt.attach)`` works)."""
        from .nn import SparseLinear

        if isinstance(module, SparseLinear):
            at = self._attached.get(module._values)
            if at is None or at.layer is not module or at.csr is not module._csr:
                self._attached[module._values] = _Attached(module)

    @torch.no_grad()
    def follow(self) -> None:
        """Moves the moments of attached layers to their weights' slots after SET or RigL
        rewrites, as the next ``step()`` would first. A captured step cannot: between a
        rewrite and its next replay (or the next capture) call this."""
        for p in self._attached:
            self._follow(p)

    def _follow(self, p) -> None:
        at = self._attached[p]
        csr = at.layer._csr
        if csr is not at.csr:
            if csr.col_indices.numel() != at.cols.numel() or csr.device == at.csr.device:
                raise RuntimeError("AdamW: an attached layer's matrix was replaced; load the "
                                   "optimizer's state and attach the layer again")
            at.snapshot()  # the layer moved to another device, with its topology
        if csr.topology_version == at.version:
            return
        if _capturing():
            raise RuntimeError("AdamW: a layer was rewritten and its moments have not followed; "
                               "call follow() (or take a step) before capturing")
        s = self.state[p]
        if s:
            names = [k for k in ("exp_avg", "exp_avg_sq") if k in s]
            states = [(s[k], s[k + "_scale"]) if k + "_scale" in s else s[k] for k in names]
            # back into the same tensors: a captured step reads them where they were
            for k, got in zip(names, carry_slots(csr.row_start, (at.cols, at.nnz),
                                                 (csr.col_indices, csr.row_nnz), states)):
                if isinstance(got, tuple):
                    s[k].copy_(got[0])
                    s[k + "_scale"].copy_(got[1])
                else:
                    s[k].copy_(got)
        at.snapshot()

    # ─── state ───

    def _init_state(self, p, group, step) -> dict:
        s = self.state[p]
        dev = p.device
        s["step"] = step
        if group["state_bits"] == 8:
            for k, dt in (("exp_avg", torch.int8), ("exp_avg_sq", torch.uint8)):
                s[k] = torch.zeros(p.shape, dtype=dt, device=dev)
                s[k + "_scale"] = torch.zeros(_blocks(p.numel()), device=dev)
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                s[k] = torch.zeros(p.shape, device=dev)
        return s

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # torch casts states to their parameter's dtype: 8-bit codes and the float32
        # moments of bfloat16 parameters are taken from the dict as they are
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            steps: dict = {}  # a count is shared within a group only, which advances it
            for i, p in zip(saved["params"], group["params"]):
                for k, v in state_dict["state"].get(i, {}).items():
                    if k == "step" and isinstance(v, torch.Tensor):
                        v = steps.setdefault((p.device, float(v)),
                                             v.detach().to(p.device, copy=True))
                    elif isinstance(v, torch.Tensor):
                        v = v.detach().to(p.device, copy=True)
                    self.state[p][k] = v
        for at in self._attached.values():
            at.snapshot()

    def _idle_counts(self, group, params) -> set:
        """Counts that parameters without a gradient stay at: those that go on leave them."""
        if len(params) == len(group["params"]):
            return set()
        return {id(self.state[p]["step"]) for p in group["params"]
                if p.grad is None and "step" in self.state.get(p, ())}

    # ─── the step ───

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            self._step_group(group)
        return loss

    def _step_group(self, group) -> None:
        capturing = _capturing()
        if capturing and not group["capturable"]:
            raise RuntimeError("AdamW: a step under graph capture needs capturable=True")
        params = [p for p in group["params"] if p.grad is not None]
        if not params:
            return
        if capturing and not all(self.state[p] for p in params):
            raise RuntimeError("AdamW: a captured step would begin the moments anew on every "
                               "replay; take one step of all its parameters before capturing")
        states, first = [], 0
        if group["capturable"] and not all(self.state[p] for p in params):
            first = torch.zeros(1, device=params[0].device)  # one count for all that begin now
        for p in params:
            if p in self._attached:
                self._follow(p)
            s = self.state[p]
            states.append(s if s else self._init_state(p, group, first))
        names = ["exp_avg", "exp_avg_sq"]
        if group["state_bits"] == 8:
            names += ["exp_avg_scale", "exp_avg_sq_scale"]
        idle = self._idle_counts(group, params) if group["capturable"] else ()
        if idle and capturing and any(id(s["step"]) in idle for s in states):
            raise RuntimeError("AdamW: a parameter that has counted along with others has no "
                               "gradient; take one such step before capturing")
        by_step: dict = {}  # more than one part only where a gradient came late or not at all
        for i, s in enumerate(states):
            if not group["capturable"]:
                s["step"] += 1
            by_step.setdefault(s["step"] if not group["capturable"] else id(s["step"]),
                               []).append(i)
        for part in by_step.values():
            if group["capturable"]:
                step = states[part[0]]["step"]
                if id(step) in idle:
                    step = step.clone()
                    for i in part:
                        states[i]["step"] = step
                step.add_(1.0)
            ps = [params[i] for i in part]
            gs = [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p in ps]
            lists = [[states[i][k] for i in part] for k in names]
            scales = tuple(lists[2:]) or None
            sizes = _check_lists(ps, gs, lists[:2], scales)
            _launch(sizes, ps, gs, lists[0], lists[1], scales, states[part[0]]["step"], group["lr"],
                    group["betas"], group["eps"], group["weight_decay"])
