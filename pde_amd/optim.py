"""The rest of a training step after the losses' backward pass: the norm of all gradients, clipping by it, AdamW.

The trainers go on with `clip_grad_norm_(parameters, max_norm); optimizer.step()`
(finetune/train_taylor_green_2d_lora_v3.py:513-516).  The functions here carry the names and arguments of
torch.nn.utils (`foreach` is taken and has no effect); each takes all tensors of the list in a few launches, with sums in
fp64, and never waits for the GPU unless `error_if_nonfinite` asks for it or a norm is handed in on the CPU.  ClippedAdamW
applies the clipping factor while it reads the gradients, so they are read twice and written never.

Tensors are float32, bfloat16 or float16 (parameters of ClippedAdamW float32 or bfloat16) on one HIP device; views into
packed buffers need no alignment beyond their type's.  Everything runs on the current stream of that device and can be
captured into a HIP graph.
"""
from __future__ import annotations

import inspect
import math
from typing import Iterable, Optional, Tuple, Union

import torch
from torch.optim.optimizer import _global_optimizer_post_hooks as _global_post_hooks, _global_optimizer_pre_hooks as _global_pre_hooks

from . import _lib

__all__ = ["get_total_norm", "clip_grad_norm_", "clip_grads_with_norm_", "ClippedAdamW"]

_ext = None


def _op():
    """the extension module with the list functions"""
    global _ext
    if _ext is None:
        _ext = _lib.optim_ext()
    return _ext


def _norm_code(norm_type) -> int:
    p = float(norm_type)
    if p not in (1.0, 2.0, math.inf):
        raise ValueError(f"pde_amd: norm_type must be 1, 2 or inf, got {norm_type!r}")
    return 0 if p == math.inf else int(p)


def _check_limit(max_norm, what: str = "max_norm") -> float:
    m = float(max_norm)
    if not m >= 0.0:
        raise ValueError(f"pde_amd: {what} must be a number >= 0, got {max_norm!r}")
    return m


def _raise_if_nonfinite(total: torch.Tensor) -> None:
    if not math.isfinite(float(total)):      # waits for the GPU
        raise RuntimeError("pde_amd: the total norm of the gradients is not finite, so they cannot be clipped by it "
                           "(error_if_nonfinite=False clips all the same)")


def get_total_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0, error_if_nonfinite: bool = False,
                   foreach: Optional[bool] = None, *, per_tensor: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """torch.nn.utils.get_total_norm: the norm of all elements of all tensors, as a 0-dim float32 tensor (whatever the
    tensors' type).  norm_type is 1, 2 or inf.  With per_tensor=True also the norm of each tensor, in one [n] tensor.
    NaN anywhere gives NaN.  No tensors: 0, on the CPU.  Tensors that are not dense in memory are copied first."""
    out = _op().total_norm(tensors, _norm_code(norm_type), bool(per_tensor))
    if error_if_nonfinite:
        _raise_if_nonfinite(out[0] if per_tensor else out)
    return out


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: Optional[bool] = None) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_: scales the gradients of all parameters in place by min(1, max_norm / (norm + 1e-6))
    and returns the norm they had, a 0-dim float32 tensor.  Parameters without a gradient are passed over.  Where the
    factor is 1 the gradients are read once and not written.  Gradients must not share memory."""
    limit, code = _check_limit(max_norm), _norm_code(norm_type)
    if not error_if_nonfinite:
        return _op().clip_grad_norm_(parameters, limit, code)
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    total = get_total_norm([p.grad for p in params if p.grad is not None], norm_type, error_if_nonfinite=True)
    _op().clip_grads_with_norm_(params, limit, total)
    return total


def clip_grads_with_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, total_norm: torch.Tensor,
                          foreach: Optional[bool] = None) -> None:
    """torch.nn.utils.clip_grads_with_norm_: the scaling of clip_grad_norm_ by a norm found elsewhere, e.g. one added up
    over the ranks that hold the other shards of the gradients.  total_norm is one value, read on the device."""
    _op().clip_grads_with_norm_(parameters, _check_limit(max_norm), total_norm)


class ClippedAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with the clipping of the gradients inside the step:

        norm = ||all gradients||_2;  c = min(1, max_norm / (norm + 1e-6));  g = c * grad
        m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2;  t = t + 1
        w = (1 - lr weight_decay) w - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    which is `clip_grad_norm_(params, max_norm); torch.optim.AdamW(...).step()` except that p.grad keeps its unclipped
    values.  max_norm=None does not clip.  After a step `total_norm` holds the norm (None where none was needed); the norm
    is over the gradients of all parameter groups.  skip_nonfinite=True leaves parameters, state and step counts as they
    are when the norm is not finite, decided on the device.  `step(total_norm=...)` takes a norm found elsewhere (added up
    over ranks) instead.

    State per parameter: 'exp_avg', 'exp_avg_sq' and, for a bfloat16 parameter, 'master' (its value in float32, from which
    the parameter is rounded at every step: write to both when changing a parameter by hand, or call `reload_masters()`),
    all float32, and the 0-dim 'step', on the device.  It is made at a parameter's first step with a gradient, and written in
    place.  Other tensors put into `state`, and state that was cleared, count from the next step on.  lr may
    be a 0-dim float32 tensor on the device, read at every step (also at every replay of a captured one).  A step can be
    captured into a graph once an eager one has run with the same parameters; keep the optimizer as long as the graph, which
    keeps the settings it was captured with and reads the gradients where they were then.  The host waits for a copy in a
    step whose parameters or state have other addresses than at the last one (the first, for instance); settings may change
    at every step without.
    """

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, max_norm: Optional[float] = None, skip_nonfinite: bool = False):
        self._plan = None
        self._captured_plans = []
        self.max_norm = None if max_norm is None else _check_limit(max_norm)
        self.skip_nonfinite = bool(skip_nonfinite)
        self.total_norm: Optional[torch.Tensor] = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def __setstate__(self, state):
        super().__setstate__(state)      # also load_state_dict comes here, with a plan that a graph may read
        for name, value in (("max_norm", None), ("skip_nonfinite", False), ("total_norm", None), ("_plan", None), ("_captured_plans", None)):
            self.__dict__.setdefault(name, value)
        self._captured_plans = self._captured_plans or []
        self._drop_plan()

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm, "skip_nonfinite": self.skip_nonfinite}

    def add_param_group(self, param_group):
        group = {**self.defaults, **param_group}
        self._hyper(group)
        if len(self.param_groups) >= 64:
            raise ValueError("pde_amd: at most 64 parameter groups")
        super().add_param_group(param_group)
        self._drop_plan()

    def _drop_plan(self) -> None:
        """The next step describes parameters and state anew; a graph goes on reading the description it was captured with."""
        if self._plan is not None and _op().adamw_captured(self._plan):
            self._captured_plans.append(self._plan)
        self._plan = None

    @staticmethod
    def _hyper(group) -> None:
        """the checks that a step makes too, ahead of the first one"""
        for name in ("amsgrad", "maximize"):      # e.g. from another optimizer's state_dict
            if group.get(name):
                raise ValueError(f"pde_amd: ClippedAdamW has no {name}")
        if float(group["weight_decay"]) != 0.0 and not group.get("decoupled_weight_decay", True):      # from torch's Adam
            raise ValueError("pde_amd: ClippedAdamW has no weight decay that is added to the gradients (decoupled_weight_decay=False)")
        lr, (b1, b2), eps, decay = group["lr"], group["betas"], float(group["eps"]), float(group["weight_decay"])
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1:
                raise ValueError(f"pde_amd: a learning rate must hold one value, got shape {tuple(lr.shape)}")
            lr = 0.0 if lr.is_cuda else float(lr)
        lr, b1, b2 = float(lr), float(b1), float(b2)
        if not (lr >= 0.0 and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0 and decay >= 0.0):
            raise ValueError(f"pde_amd: need lr >= 0, 0 <= betas < 1, eps >= 0 and weight_decay >= 0, got lr={lr}, betas=({b1}, {b2}), "
                             f"eps={eps}, weight_decay={decay}")

    @torch.no_grad()
    def _make_state(self, params) -> None:
        """zeros for parameters that see their first gradient; their step counts lie side by side"""
        if not params:
            return
        if params[0].is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pde_amd: an optimizer's first step cannot be captured into a graph: run one step before")
        steps = torch.zeros(len(params), dtype=torch.float32, device=params[0].device)
        for i, p in enumerate(params):
            state = dict(step=steps[i], exp_avg=torch.zeros_like(p, dtype=torch.float32, requires_grad=False),
                         exp_avg_sq=torch.zeros_like(p, dtype=torch.float32, requires_grad=False))
            if p.dtype == torch.bfloat16:
                state["master"] = p.detach().float()
            self.state[p] = state

    def _build(self):
        params = [p for group in self.param_groups for p in group["params"]]
        groups = [g for g, group in enumerate(self.param_groups) for _ in group["params"]]
        index = [i for i, p in enumerate(params) if self.state.get(p)]
        states = [self.state[params[i]] for i in index]
        for i, s in zip(index, states):
            need = {"step", "exp_avg", "exp_avg_sq"} | ({"master"} if params[i].dtype == torch.bfloat16 else set())
            if not need <= set(s):
                raise ValueError(f"pde_amd: the state of a parameter must hold {sorted(need)}, got {sorted(s)}")
        return _op().adamw_plan(
            params, groups, index, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
            [s.get("master", s["exp_avg"]) for s in states], [s["step"] for s in states])

    def step(self, *args, **kwargs):
        """step(closure=None, *, total_norm=None): one update of every parameter that has a gradient; returns the closure's
        loss, if one is given."""
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_pre_hooks or _global_post_hooks:
            if type(self).step is ClippedAdamW.step:      # the base class wraps a subclass's own step, with the hooks
                return self._step_with_hooks(*args, **kwargs)
        return self._step(*args, **kwargs)

    # Says that step() runs the hooks itself.  The base class would wrap it otherwise, and the wrapper's profiler range takes
    # 7 us of the host's time, as much as a small step takes on the GPU.
    step.hooked = True

    def _step_with_hooks(*args, **kwargs):
        """torch's hooks: they get the call's arguments with the optimizer first, and the ahead ones may change them"""
        self = args[0]
        for hook in (*_global_pre_hooks.values(), *self._optimizer_step_pre_hooks.values()):
            changed = hook(self, args, kwargs)
            if changed is not None:
                if not isinstance(changed, tuple) or len(changed) != 2:
                    raise RuntimeError(f"pde_amd: a step's pre-hook must return None or a tuple of (new_args, new_kwargs), but got {changed!r}")
                args, kwargs = changed
        loss = type(self)._step(*args, **kwargs)
        for hook in (*self._optimizer_step_post_hooks.values(), *_global_post_hooks.values()):
            hook(self, args, kwargs)
        return loss

    def _step(self, closure=None, *, total_norm: Optional[torch.Tensor] = None):
        if total_norm is not None and not isinstance(total_norm, torch.Tensor):
            raise TypeError(f"pde_amd: total_norm must be a tensor, got {type(total_norm).__name__}")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        limit = -1.0 if self.max_norm is None else _check_limit(self.max_norm)
        skip = bool(self.skip_nonfinite)
        norm = False if self._plan is None else _op().adamw_step(self._plan, self.param_groups, limit, skip, total_norm, self.state)
        if norm is False:      # no plan yet, or one of other parameters
            for group in self.param_groups:
                self._hyper(group)
            self._drop_plan()
            self._plan = self._build()
            norm = _op().adamw_step(self._plan, self.param_groups, limit, skip, total_norm, self.state)
        if isinstance(norm, list):      # parameters that see their first gradient
            params = [p for group in self.param_groups for p in group["params"]]
            self._make_state([params[i] for i in norm])
            self._drop_plan()
            self._plan = self._build()
            norm = _op().adamw_step(self._plan, self.param_groups, limit, skip, total_norm, self.state)
        if norm is False or isinstance(norm, list):
            raise RuntimeError("pde_amd: parameters or state of the optimizer changed during its step")
        self.total_norm = total_norm if norm is None else norm
        return loss

    step.__signature__ = inspect.signature(_step)

    @torch.no_grad()
    def reload_masters(self) -> None:
        """Take the float32 values of the bfloat16 parameters from the parameters again, after these were written by hand."""
        for p, s in self.state.items():
            if "master" in s:
                s["master"].copy_(p)

    def load_state_dict(self, state_dict) -> None:
        """As torch.optim.Optimizer's, but all state stays float32 (there it takes the parameter's type) in the
        parameter's layout, in tensors of the optimizer's own.  Once a step has been captured it goes into the tensors that are
        there already, with which the graph goes on: take a deep copy of a state_dict() that is to outlive such a load."""
        before, used = dict(self.state), []

        def last_pre_hook(_, loaded):
            self._check_state(loaded)
            used.append(loaded)

        # behind the other pre-hooks and ahead of the other post-hooks: what the former return is loaded, and what the latter
        # set stays
        pre = self.register_load_state_dict_pre_hook(last_pre_hook)
        post = self.register_load_state_dict_post_hook(lambda _: self._take_state(used[-1], before), prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            pre.remove()
            post.remove()

    def _given_state(self, loaded):
        """(parameter, its entry) of every parameter that has state in a state_dict"""
        saved = [i for g in loaded["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        return [(p, loaded["state"][i]) for i, p in zip(saved, params) if loaded["state"].get(i)]

    def _check_state(self, loaded) -> None:
        if [len(g["params"]) for g in loaded["param_groups"]] != [len(g["params"]) for g in self.param_groups]:
            return      # the base class refuses it
        for p, given in self._given_state(loaded):
            for name in ("exp_avg", "exp_avg_sq", "master"):
                value = given.get(name, p)
                if not isinstance(value, torch.Tensor) or value.shape != p.shape:
                    got = f"shape {tuple(value.shape)}" if isinstance(value, torch.Tensor) else type(value).__name__
                    raise ValueError(f"pde_amd: state {name!r} must have its parameter's shape {tuple(p.shape)}, got {got}")
            step = given.get("step", 0)
            try:
                one = torch.as_tensor(step).numel() == 1
            except (TypeError, ValueError, RuntimeError):
                one = False
            if not one:
                raise ValueError(f"pde_amd: state 'step' must be one number, got {step!r}")

    @torch.no_grad()
    def _take_state(self, loaded, before) -> None:
        """the state of a state_dict, which the base class has taken already, once more from its own values"""
        given_state, in_place = self._given_state(loaded), bool(self._captured_plans)
        written = [t for s in before.values() for t in s.values() if isinstance(t, torch.Tensor)] if in_place else []
        written = {t.untyped_storage().data_ptr() for t in written}

        def source(value):
            value = torch.as_tensor(value).detach()
            return value.clone() if value.layout is torch.strided and value.untyped_storage().data_ptr() in written else value

        # all sources ahead of the first write: some may lie in the tensors that are written
        taken = [{name: source(value) for name, value in given.items() if name in ("step", "exp_avg", "exp_avg_sq", "master")} for _, given in given_state]
        for (p, _), values in zip(given_state, taken):
            state, there = dict(self.state[p]), before.get(p) or {}      # entries of the user's as the base class took them
            if p.dtype == torch.bfloat16:
                values.setdefault("master", p.detach())
            for name, value in values.items():
                like = torch.empty((), device=p.device) if name == "step" else p
                t = there.get(name) if in_place else None
                if t is None or t.shape != like.shape or t.device != p.device or t.dtype != torch.float32 or t.stride() != like.stride():
                    t = torch.empty_like(like, dtype=torch.float32, requires_grad=False)
                state[name] = t.copy_(value.reshape(like.shape))
            self.state[p] = state
