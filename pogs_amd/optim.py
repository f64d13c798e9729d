"""Fused Adam over parameter groups on MI355X: the optimiser step of the POGS trainer.

Mirrors nerfstudio's ``Optimizers`` as the trainer drives it
(``nerfstudio/engine/optimizers.py:74-193``, ``nerfstudio/engine/trainer.py:494-510``) for the configuration
POGS uses (``pogs/pogs_config.py:27,38-85``): one ``torch.optim.Adam(lr, eps=1e-15)`` per named group, an
optional exponential-decay schedule per group (``nerfstudio/engine/schedulers.py:92-141``) and per-group
gradient-accumulation periods.  Same method names and meaning; the difference is that all groups due in an
iteration are updated by ONE kernel launch (``pr_adam_step``).  No PyTorch fallback.

Gradient clipping (``OptimizerConfig.max_norm``, applied in ``optimizers.py:159-172`` through
``torch.nn.utils.clip_grad_norm_``): a group whose config has ``max_norm`` is clipped to that norm in its step, by a factor
that the Adam kernel takes from device memory, so clipping costs one pass over the gradients and no host
synchronisation.  ``grad_norm`` and ``clip_grad_norm_`` are the same kernels for callers with an optimiser of their own.

State is kept in torch's own layout, so ``state_dict()[name]`` loads into ``torch.optim.Adam`` and back.
"""
from __future__ import annotations

import ctypes
import math
import struct
from array import array
from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from .rendering import _call, _on, _raw_stream, _refuse_dual


_ADAM_GROUP = struct.Struct("=4Q2q4d")     # pr_adam_group
_CLIP_RULE = struct.Struct("=2id")          # pr_clip_rule
_GRAD_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}        # PR_F32, PR_F16, PR_BF16
_NORM_KINDS = {1.0: 1, 2.0: 2, math.inf: 3}                                   # PR_NORM_1, PR_NORM_2, PR_NORM_INF


def _one_block(t: Tensor) -> bool:
    """Whether the elements of ``t`` fill one block of memory, in any order of dimensions."""
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _grad_table(grads: Sequence[Tensor]) -> array:
    """The grads as an array of ``pr_grad_tensor``: pointer, elements, type and (in the upper half word) set 0."""
    words = array("q", bytes(24 * len(grads)))
    words[0::3] = array("q", [g.data_ptr() for g in grads])
    words[1::3] = array("q", [g.numel() for g in grads])
    words[2::3] = array("q", [_GRAD_TYPES[g.dtype] for g in grads])
    return words


def _address(a: array) -> ctypes.c_void_p:
    return ctypes.c_void_p(a.buffer_info()[0])


def _norm_buffers(nbytes: int, shape: tuple, device) -> Tuple[Tensor, Tensor]:
    return (torch.empty(max(nbytes // 8, 1), dtype=torch.float64, device=device),
            torch.empty(shape, dtype=torch.float32, device=device))


def _check_grads(grads: Sequence[Tensor]) -> torch.device:
    if {g.layout for g in grads} != {torch.strided} or not all([g.is_cuda for g in grads]):
        raise RuntimeError("pogs_amd.optim needs dense gradients on a HIP device (no CPU fallback)")
    for t in {g.dtype for g in grads}:
        if t not in _GRAD_TYPES:
            raise TypeError(f"gradients must be float32, float16 or bfloat16, got {t}")
    devices = {g.device for g in grads}
    if len(devices) > 1:
        raise RuntimeError(f"gradients are on different devices: {sorted(map(str, devices))}")
    return devices.pop()


def _flat(grads: List[Tensor]) -> List[Tensor]:
    """The gradients as blocks of memory: themselves, or a copy of one whose elements are scattered."""
    if all([g.is_contiguous() for g in grads]):
        return grads
    return [g if g.is_contiguous() or _one_block(g) else g.detach().contiguous() for g in grads]


def _norm_kind(norm_type: float) -> int:
    kind = _NORM_KINDS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type}")
    return kind


def _max_norm(value) -> float:
    value = float(value)
    if not value >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {value}")
    return value


def grad_norm(tensors: Union[Tensor, Iterable[Tensor]], norm_type: float = 2.0) -> Tensor:
    """Norm over all elements of all ``tensors`` (gradients; float32, float16 or bfloat16 in any mix and layout) as a
    0-d float32 tensor on their device.  Counterpart of ``torch.nn.utils.get_total_norm`` for ``norm_type`` 1, 2 and inf.
    Sums are kept in float64, in an order that depends on the sizes alone: equal inputs give equal bits.  No host
    synchronisation; safe in a captured graph.  A plain number to autograd, as in torch; forward-mode tensors are refused.
    An empty list has norm 0 (on the CPU, as in torch)."""
    kind = _norm_kind(norm_type)
    grads = [tensors] if isinstance(tensors, Tensor) else list(tensors)
    if not grads:
        return torch.tensor(0.0)
    _refuse_dual("grad_norm", grads)
    dev = _check_grads(grads)
    lib = _lib.load()
    with _on(dev):
        flat = _flat(grads)
        table = _grad_table(flat)
        at, n = _address(table), len(flat)
        nbytes = lib.pr_grad_norm_scratch_bytes(at, n, 1)
        scratch, norm = _norm_buffers(nbytes, (), dev)
        _call("pr_grad_norm", at, n, 1, kind, scratch.data_ptr(), nbytes, norm.data_ptr(),
              _raw_stream(dev.index))
    return norm


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> Tensor:
    """``torch.nn.utils.clip_grad_norm_``: multiplies the ``.grad`` of every parameter that has one by
    ``min(1, max_norm / (norm + 1e-6))``, in place, and returns the norm over all of them before that (0-d float32).

    Gradients may be float32, float16 or bfloat16, of any layout, all on one device and in memory of their own: two that
    begin at the same place (a parameter listed twice) or whose blocks overlap are refused, as scaling them at once is a
    race, and so is an expanded one; then nothing has been scaled.  Each value is rounded once, to its own type.  Where the norm is within bounds no gradient is written.  A norm that is not finite
    gives what torch gives: factor 0 for an infinite norm, NaN for a NaN one; ``error_if_nonfinite`` raises instead, and
    only then does the host wait for the device."""
    kind, max_norm = _norm_kind(norm_type), _max_norm(max_norm)
    params = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    grads = [g for p in params if (g := p.grad) is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite and not math.isfinite(grad_norm(grads, norm_type).item()):
        raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is non-finite, so it "
                           "cannot be clipped. To disable this error and scale the gradients by the non-finite norm "
                           "anyway, set `error_if_nonfinite=False`")
    dev, lib = _check_grads(grads), _lib.load()
    with _on(dev):
        flat = _flat(grads)
        if flat is not grads:      # a copy shares nothing, so the blocks' own check would miss it
            starts = [g.data_ptr() for g in grads if g.numel()]
            if len(set(starts)) < len(starts):
                raise RuntimeError("clip_grad_norm_: two gradients share memory")
            if any([0 in g.stride() and any(st == 0 and n > 1 for st, n in zip(g.stride(), g.shape)) for g in grads]):
                raise RuntimeError("clip_grad_norm_: an expanded gradient cannot be scaled in place")
        table, limit = _grad_table(flat), ctypes.c_double(max_norm)
        at, n = _address(table), len(flat)
        nbytes = lib.pr_grad_norm_scratch_bytes(at, n, 1)
        scratch, norm = _norm_buffers(nbytes, (), dev)
        _call("pr_grad_clip", at, n, 1, kind, ctypes.addressof(limit), scratch.data_ptr(), nbytes, norm.data_ptr(),
              _raw_stream(dev.index))
        torch.autograd.graph.increment_version(flat)     # written in place, as far as autograd is concerned too
        if flat is not grads:
            with torch.no_grad():
                for g, f in zip(grads, flat):
                    if f is not g:
                        g.copy_(f)
    return norm


class ExponentialDecay:
    """Learning-rate multiplier of ``ExponentialDecayScheduler`` (``schedulers.py:116-141``): optional warm-up
    from ``lr_pre_warmup``, then log-linear interpolation from ``lr_init`` to ``lr_final`` over ``max_steps``."""

    def __init__(self, lr_final: Optional[float] = None, max_steps: int = 100000, warmup_steps: int = 0,
                 lr_pre_warmup: float = 1e-8, ramp: str = "cosine"):
        self.lr_final, self.max_steps, self.warmup_steps = lr_final, max_steps, warmup_steps
        self.lr_pre_warmup, self.ramp = lr_pre_warmup, ramp

    def lr(self, lr_init: float, step: int) -> float:
        lr_final = lr_init if self.lr_final is None else self.lr_final
        if step < self.warmup_steps:
            if self.ramp == "cosine":
                return self.lr_pre_warmup + (lr_init - self.lr_pre_warmup) * math.sin(
                    0.5 * math.pi * min(max(step / self.warmup_steps, 0.0), 1.0))
            return self.lr_pre_warmup + (lr_init - self.lr_pre_warmup) * step / self.warmup_steps
        t = min(max((step - self.warmup_steps) / (self.max_steps - self.warmup_steps), 0.0), 1.0)
        return math.exp(math.log(lr_init) * (1 - t) + math.log(lr_final) * t)


class Optimizers:
    """config: ``{group: {"lr": float, "eps": float = 1e-15, "betas": (0.9, 0.999), "scheduler": ExponentialDecay
    or None, "max_norm": float or None}}``; param_groups: ``{group: [parameters]}`` (float32 HIP tensors).

    ``max_norm``: the group's gradient, over all its parameters, is clipped to that 2-norm in every step, as by
    ``clip_grad_norm_``; the parameters' ``.grad`` keep their values.  ``grad_norms`` holds the norms that the last step
    clipped by."""

    def __init__(self, config: Dict[str, dict], param_groups: Dict[str, List[Tensor]]):
        _lib.load()
        self.config, self.parameters = config, {}
        self._state: Dict[str, List[dict]] = {}
        self._sched_steps: Dict[str, int] = {}
        self._norms: List[Tuple[Tensor, Dict[str, int]]] = []      # of the last step: norms, place of each group
        self._norm_of: Optional[Dict[str, Tensor]] = None          # made from them when asked for
        for name, params in param_groups.items():
            if name not in config:
                raise RuntimeError(f"Optimizer config for '{name}' not found in config file. Provided configs "
                                   f"were: {config.keys()}")
            for p in params:
                if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
                    raise RuntimeError("pogs_amd.optim needs contiguous float32 parameters on a HIP device "
                                       "(no CPU fallback)")
            if config[name].get("max_norm") is not None:
                _max_norm(config[name]["max_norm"])
            self.parameters[name] = list(params)
            self._state[name] = [{} for _ in params]
            self._sched_steps[name] = 0

    # ---- learning rates ------------------------------------------------------------------------------------
    def lr(self, name: str) -> float:
        cfg = self.config[name]
        sched = cfg.get("scheduler")
        return cfg["lr"] if sched is None else sched.lr(cfg["lr"], self._sched_steps[name])

    def scheduler_step(self, name: str) -> None:
        if self.config[name].get("scheduler") is not None:
            self._sched_steps[name] += 1

    def scheduler_step_all(self, step: int) -> None:
        for name in self.parameters:
            self.scheduler_step(name)

    # ---- gradients -----------------------------------------------------------------------------------------
    def zero_grad_all(self) -> None:
        self.zero_grad_some(list(self.parameters))

    def zero_grad_some(self, param_groups: List[str]) -> None:
        for name in param_groups:
            for p in self.parameters[name]:
                p.grad = None

    # ---- steps ---------------------------------------------------------------------------------------------
    def optimizer_step(self, param_group_name: str) -> None:
        self.optimizer_step_some([param_group_name])

    def optimizer_step_all(self, max_norm: Optional[float] = None) -> None:
        self.optimizer_step_some(list(self.parameters), max_norm)

    def optimizer_step_some(self, param_groups: Iterable[str], max_norm: Optional[float] = None) -> None:
        """One Adam update of every parameter (that has a gradient) of the named groups, in one launch per
        ``pr_adam_max_groups()`` tensors.  Groups with a ``max_norm`` of their own are clipped one by one; ``max_norm``
        given here clips the gradient of all the named groups together to one norm instead, and then none of them may
        have its own."""
        param_groups = list(param_groups)        # gone through more than once
        limits = [self.config[name].get("max_norm") for name in param_groups]
        if max_norm is not None:
            max_norm = _max_norm(max_norm)
            if any(m is not None for m in limits):
                raise ValueError("a max_norm over all groups and a max_norm of a group's own exclude each other")
        if max_norm is not None or any(m is not None for m in limits):
            limits = self._check_clipped(param_groups, limits)       # before any state is touched
        entries, rules, keep, stepped = [], [], [], []     # rules: (group or None for all together, its limit or None)
        for name, limit in zip(param_groups, limits):
            cfg = self.config[name]
            b1, b2 = cfg.get("betas", (0.9, 0.999))
            lr, eps = self.lr(name), cfg.get("eps", 1e-15)
            for p, st in zip(self.parameters[name], self._state[name]):
                if p.grad is None:
                    continue
                g = p.grad
                if g.dtype != torch.float32 or not g.is_contiguous() or g.data_ptr() % 16:
                    g = g.float().contiguous().clone()
                if not st:
                    st["step"] = 0
                    st["exp_avg"] = torch.zeros_like(p)
                    st["exp_avg_sq"] = torch.zeros_like(p)
                st["step"] += 1
                rules.append((None, max_norm) if max_norm is not None else (name, limit))
                keep.append(g)
                stepped.append(p)
                entries.append(_ADAM_GROUP.pack(p.data_ptr(), g.data_ptr(), st["exp_avg"].data_ptr(),
                                                st["exp_avg_sq"].data_ptr(), p.numel(), st["step"], lr, b1, b2, eps))
        self._norms, self._norm_of = [], None
        if not entries:
            return
        dev = keep[0].device
        with _on(dev):
            if all(limit is None for _, limit in rules):
                chunk = _lib.load().pr_adam_max_groups()
                for i in range(0, len(entries), chunk):
                    part = entries[i:i + chunk]
                    _call("pr_adam_step", b"".join(part), len(part), _raw_stream(dev.index))
            else:
                self._step_clipped(entries, rules, param_groups, dev, _raw_stream(dev.index))
        torch.autograd.graph.increment_version(stepped)     # written in place: a graph that saved one is refused
        del keep

    def _check_clipped(self, param_groups: List[str], limits: list) -> List[Optional[float]]:
        """The groups' limits.  A parameter that is there twice would count twice in the norm and be stepped by two
        workgroups at once; a norm is taken on one device."""
        params = [p for name in param_groups for p in self.parameters[name]]
        if len(set(map(id, params))) < len(params):
            raise ValueError("a clipped step takes every parameter once: a group or a parameter is listed twice")
        if len({p.get_device() for p in params}) > 1 and len({p.get_device() for p in params if p.grad is not None}) > 1:
            raise RuntimeError("a clipped step takes parameters of one device: step the groups of each device on their own")
        return [None if m is None else _max_norm(m) for m in limits]

    def _step_clipped(self, entries: List[bytes], rules: list, param_groups: List[str], device, stream: int) -> None:
        """The step where a group at least has a limit, for as many norms at once as a call takes."""
        lib = _lib.load()
        most, i = lib.pr_grad_norm_max_sets(), 0
        while i < len(entries):
            of, clips, lo = {}, [], i
            for name, limit in rules[i:]:
                if limit is not None and name not in of:
                    if len(of) == most:
                        break
                    of[name] = len(of)
                clips.append(_CLIP_RULE.pack(-1, 0, 0.0) if limit is None else _CLIP_RULE.pack(of[name], 0, limit))
            i = lo + len(clips)
            groups, by, n, sets = b"".join(entries[lo:i]), b"".join(clips), len(clips), max(len(of), 1)
            nbytes = lib.pr_adam_clip_scratch_bytes(groups, by, n, sets)
            scratch, norms = _norm_buffers(nbytes, (sets,), device)
            _call("pr_adam_step_clipped", groups, by, n, sets, scratch.data_ptr(), nbytes, norms.data_ptr(), stream)
            self._norms.append((norms, {g: 0 for g in param_groups} if None in of else of))

    @property
    def grad_norms(self) -> Dict[str, Tensor]:
        """The norms that the last step clipped by, one 0-d tensor on the device for each group."""
        if self._norm_of is None:
            self._norm_of = {}
            for norms, of in self._norms:
                each = norms.unbind()
                self._norm_of.update((name, each[i]) for name, i in of.items())
        return self._norm_of

    def state(self, name: str, index: int = 0) -> dict:
        """The Adam state of one parameter of a group (``step``, ``exp_avg``, ``exp_avg_sq``; empty before its first
        step).  The tensors are the live ones."""
        return self._state[name][index]

    # the trainer's per-iteration bookkeeping (trainer.py:494-510)
    @staticmethod
    def groups_to_zero(step: int, names, accumulation: Dict[str, int]) -> List[str]:
        return [n for n in names if step % accumulation.get(n, 1) == 0]

    @staticmethod
    def groups_to_step(step: int, names, accumulation: Dict[str, int]) -> List[str]:
        return [n for n in names if step % accumulation.get(n, 1) == accumulation.get(n, 1) - 1]

    # ---- checkpoints: torch.optim.Adam's own layout ----------------------------------------------------------
    def state_dict(self) -> Dict[str, dict]:
        out = {}
        for name, params in self.parameters.items():
            cfg = self.config[name]
            state = {i: {"step": torch.tensor(float(st["step"])), "exp_avg": st["exp_avg"],
                         "exp_avg_sq": st["exp_avg_sq"]}
                     for i, st in enumerate(self._state[name]) if st}
            group = {"lr": self.lr(name), "betas": tuple(cfg.get("betas", (0.9, 0.999))), "eps": cfg.get("eps", 1e-15),
                     "weight_decay": 0, "amsgrad": False, "maximize": False, "foreach": None, "capturable": False,
                     "differentiable": False, "fused": None, "decoupled_weight_decay": False,
                     "initial_lr": cfg["lr"], "params": list(range(len(params)))}
            out[name] = {"state": state, "param_groups": [group]}
        return out

    def load_optimizers(self, loaded_state: Dict[str, dict]) -> None:
        for name, sd in loaded_state.items():
            for i, st in sd["state"].items():
                p = self.parameters[name][int(i)]
                self._state[name][int(i)] = {
                    "step": int(float(st["step"])),
                    "exp_avg": st["exp_avg"].to(p.device, torch.float32).contiguous().clone(),
                    "exp_avg_sq": st["exp_avg_sq"].to(p.device, torch.float32).contiguous().clone()}
