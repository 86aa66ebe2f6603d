"""The step behind a LoRA training step's backward pass, over every factor in a few launches: ``clip_grad_norm_`` and AdamW,
the two lines that the reference's trainer takes from torch (``train_t2i_lora_cached.py:329-332``).

:class:`AdamW` keeps its moments in 32 bits, or in 8 bits with a scale for every 256 elements: 2 bytes for an element in
place of 8, and 16 bytes moved by a step in place of 28.  A group's moments lie in flat buffers, each parameter's at a
multiple of 256 elements; ``state[p]`` holds views of them.  What is put in their place, or taken out, counts: the next step
lays the group's moments out anew from what ``state`` says, zeros where it says nothing.
"""
from __future__ import annotations

import importlib
import inspect
import math
from types import SimpleNamespace

import torch

from . import _lib

_BLOCK = _lib.MOMENT_BLOCK

# what torch.optim.optimizer.register_optimizer_step_pre_hook and its post form register, for every optimizer
_torch_optimizer = importlib.import_module("torch.optim.optimizer")
_EVERY = (_torch_optimizer._global_optimizer_pre_hooks, _torch_optimizer._global_optimizer_post_hooks)


def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Scale the gradients of ``parameters`` (a tensor, or an iterable of them) in place so that their 2-norm, taken over all
    together, is at most ``max_norm``: ``torch.nn.utils.clip_grad_norm_`` of the 2-norm.  Returns the norm before, a float32
    tensor on the gradients' device (nothing waits for it).  The factor is ``min(1, max_norm / (norm + 1e-6))`` and each
    gradient is rounded once; a norm that is infinite or NaN gives the gradients that torch's gives."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be 0 or above, got {max_norm}")
    out = _lib.grad_norm(params, max_norm, True)
    return torch.zeros(()) if out is None else out[0]


class AdamW(torch.optim.Optimizer):
    """AdamW (Loshchilov and Hutter, "Decoupled weight decay regularization", 2019) with the update of ``torch.optim.AdamW``,
    in float32, over contiguous parameters in float32, bfloat16 or float16 whose gradients have their type.

    ``max_norm``: the gradients, over all groups together, are first brought to this 2-norm at most, as ``clip_grad_norm_``
    does it, but they are not written: the step multiplies them as it reads them.  :attr:`grad_norm` holds the norm of the
    last step.  A norm that is infinite or NaN skips the step on the device: parameters, moments and counts stay.

    ``state_bits=8``: the first moment in e4m3, the root of the second in 4 bits of exponent and 4 of fraction, both scaled
    by the largest of 256 neighbours.  ``stochastic=True`` rounds bfloat16 parameters to one of their two neighbours at
    random instead of to the nearest, so that updates below half a step are not lost (the reference's full fine-tune does
    that, ``fused_adamw.py:44-56``).  Codes and such parameters are rounded by chance, with bits that are a function of
    ``seed``, the step and the element's place in its group: equal runs give equal results.  Groups with one seed share
    those bits place by place; each may have its own.

    ``lr`` may be a float32 tensor of one element on the device (read there, for captured graphs).  Without ``max_norm``, a
    gradient that is infinite or NaN spoils its own element, as in torch.  Make a step, or load a state, before a graph
    capture: the moments are made at the first."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 max_norm: float | None = None, state_bits: int = 32, stochastic: bool = False, seed: int = 0):
        defaults = {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay, "state_bits": state_bits,
                    "stochastic": stochastic, "seed": seed}
        if max_norm is not None and not float(max_norm) >= 0:
            raise ValueError(f"max_norm must be 0 or above, got {max_norm}")
        self.max_norm = None if max_norm is None else float(max_norm)
        self.grad_norm = None
        self._held = {}         # id of a group's list of parameters -> its moments' buffers (which hold the list)
        self._seen = None       # the state's keys, its values and theirs, as they were last found to be those buffers'
        super().__init__(params, defaults)

    def add_param_group(self, param_group: dict) -> None:
        for name, value in self.defaults.items():
            param_group.setdefault(name, value)
        _check_options(param_group)
        super().add_param_group(param_group)

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm}

    def __setstate__(self, state) -> None:
        self.__dict__.setdefault("max_norm", None)
        self.grad_norm, self._held, self._seen = None, {}, None       # laid out again from the states at the next step
        super().__setstate__(state)
        for group in self.param_groups:
            for name, value in self.defaults.items():
                group.setdefault(name, value)
            _check_options(group)

    # -- moments -------------------------------------------------------------------------------------------------
    def _moments_of(self, group: dict) -> SimpleNamespace:
        """A group's buffers, made when they are not there: zeros, or the states that its parameters have."""
        params = group["params"]
        held = self._held.get(id(params))
        # a list that grew or shrank is refused by the step; one with others in it, or in other bits, is laid out anew
        if held is not None and (len(params) != len(held.of) or
                                 held.bits == group["state_bits"] and _lib.same_items(params, held.of)):
            return held
        devices = {p.device for p in params}
        if len(devices) != 1 or next(iter(devices)).type != "cuda":
            raise RuntimeError(f"k2q kernels need a group's parameters on one gfx950 GPU, got {sorted(map(str, devices))}")
        dev = next(iter(devices))
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the moments are not made yet and a graph capture would make them at every replay: make a "
                               "step, or load a state, before it")
        for k, p in enumerate(params):
            if p.dtype not in _lib.STEP_DTYPES:
                raise ValueError(f"parameter {k} is {p.dtype}, not one of {_lib.STEP_DTYPES}")
            _check_state(self.state.get(p) or None, p, group["state_bits"])
        starts, total = [], 0
        for p in params:
            starts.append(total)
            total += -(-p.numel() // _BLOCK) * _BLOCK
        held = SimpleNamespace(params=params, of=list(params), bits=group["state_bits"], starts=starts, states=[],
                               steps=torch.zeros(len(params), device=dev))
        kinds = _kinds(held.bits)
        for name, (dtype, per) in kinds.items():
            setattr(held, name, torch.zeros(total // per, device=dev, dtype=torch.uint8).view(dtype)
                    if dtype.itemsize == 1 else torch.zeros(total // per, device=dev, dtype=dtype))
        with torch.no_grad():
            for k, (p, start) in enumerate(zip(params, starts)):
                old, new = self.state.get(p), {"step": held.steps[k]}
                for name, (dtype, per) in kinds.items():
                    flat = getattr(held, name)
                    new[name] = flat[start:start + p.numel()].view(p.shape) if per == 1 else \
                        flat[start // per:start // per - (-p.numel() // per)]
                if old:
                    for name, view in new.items():
                        _copy(view, old[name])
                self.state[p] = new
                held.states.append((new, list(new.values())))
        self._held[id(params)] = held
        self._note_state()
        return held

    def _note_state(self) -> None:
        dicts = list(self.state.values())
        self._seen = (list(self.state), dicts, [v for d in dicts if isinstance(d, dict) for v in d.values()])

    def _follow_state(self) -> None:
        """Drop the buffers of groups whose states are not theirs any more: the next use makes them from the states."""
        if self._seen is not None and _lib.unchanged(self.state, *self._seen):
            return
        for key, held in list(self._held.items()):
            if not all(self.state.get(p) is d and _lib.same_items(list(d.values()), views)
                       for p, (d, views) in zip(held.of, held.states)):
                del self._held[key]
        self._note_state()

    def moments(self, group: int = 0, dtype: torch.dtype = torch.float32):
        """``(exp_avg, exp_avg_sq)`` of a group's parameters as numbers, flat, each parameter's from a multiple of 256
        elements on: its own buffers where they are held in ``dtype``, else what they hold in ``dtype`` (float32 or
        bfloat16)."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"dtype must be float32 or bfloat16, got {dtype}")
        self._follow_state()
        held = self._moments_of(self.param_groups[group])
        if held.bits == 32 or not held.exp_avg.numel():
            return held.exp_avg.to(dtype), held.exp_avg_sq.to(dtype)
        return _lib.moments(held.exp_avg, held.exp_avg_scale, held.exp_avg_sq, held.exp_avg_sq_scale, dtype)

    def load_state_dict(self, state_dict: dict) -> None:
        """A state of this class, or, in 32 bits, of ``torch.optim.AdamW`` (without ``amsgrad`` or ``maximize``).  The values
        are copied, in their own types."""
        saved, states = state_dict["param_groups"], state_dict["state"]
        # options that a state does not name stay; what does not fit is refused before anything changes
        own = [{k: g[k] for k in self.defaults} for g in self.param_groups]
        saved = [{**g, **s} for g, s in zip(own, saved)] + saved[len(own):]
        for s, g in zip(saved, self.param_groups):
            _check_options(s)
            for n, p in zip(s["params"], g["params"]):
                _check_state(states.get(n), p, s["state_bits"])
        super().load_state_dict({**state_dict, "state": {}, "param_groups": saved})
        for s, g in zip(saved, self.param_groups):
            for n, p in zip(s["params"], g["params"]):
                if n in states:
                    self.state[p] = dict(states[n])
            if any(p in self.state for p in g["params"]):
                self._moments_of(g)

    # -- the step ------------------------------------------------------------------------------------------------
    def step(self, *args, **kwargs):
        """``step(closure=None)``: one step of every parameter that has a gradient; ``closure``, if given, is called first and
        its value returned."""
        if torch.autograd._profiler_enabled():
            with torch.autograd.profiler.record_function("Optimizer.step#AdamW.step"):
                return self._hooked((self, *args), kwargs)
        return self._hooked((self, *args), kwargs)

    def _hooked(self, args: tuple, kwargs: dict):
        """A step between its hooks, which get what torch gives them: the arguments with the optimizer ahead; those in front may
        return others."""
        for hook in [*_EVERY[0].values(), *self._optimizer_step_pre_hooks.values()]:
            given = hook(self, args, kwargs)
            if given is not None:
                if not (isinstance(given, tuple) and len(given) == 2):
                    raise RuntimeError(f"a hook ahead of a step must return None or a tuple (args, kwargs), got {given!r}")
                args, kwargs = given
        loss = AdamW._closure_and_step(*args, **kwargs)
        for hook in [*self._optimizer_step_post_hooks.values(), *_EVERY[1].values()]:
            hook(self, args, kwargs)
        return loss

    def _closure_and_step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._step()
        return loss

    step.__signature__ = inspect.signature(_closure_and_step)
    step.hooked = True      # hooks and the profiler's label are above: torch's own wrapper takes 12 of a small step's 28 us

    def _step(self) -> None:
        groups, squares, norm = self.param_groups, None, None
        self._follow_state()
        if self.max_norm is not None and len(groups) > 1:       # of one group, the step's own call takes it
            squares = _lib.grad_norm([p for g in groups for p in g["params"]], self.max_norm, False)
            if squares is not None:
                norm = torch.empty(2, device=squares.device)
        for g in groups:
            if not g["params"]:
                continue
            held = self._moments_of(g)
            lr, lr_of = g["lr"], None
            if isinstance(lr, torch.Tensor):
                lr, lr_of = (0.0, lr) if lr.is_cuda else (float(lr), None)
            scales = (held.exp_avg_scale, held.exp_avg_sq_scale) if held.bits == 8 else (None, None)
            out = _lib.adamw(g["params"], held.starts, held.bits, held.exp_avg, held.exp_avg_sq, *scales, held.steps, lr,
                             lr_of, *g["betas"], g["eps"], g["weight_decay"], squares, self.max_norm, norm, g["stochastic"],
                             g["seed"])
            norm = out if len(groups) == 1 else norm
        self.grad_norm = None if norm is None else norm[0]


def _kinds(bits: int) -> dict:
    """A parameter's states but the count of steps: (type, elements that share one)."""
    if bits == 32:
        return {"exp_avg": (torch.float32, 1), "exp_avg_sq": (torch.float32, 1)}
    return {"exp_avg": (torch.float8_e4m3fn, 1), "exp_avg_sq": (torch.uint8, 1), "exp_avg_scale": (torch.float32, _BLOCK),
            "exp_avg_sq_scale": (torch.float32, _BLOCK)}


def _copy(view: torch.Tensor, value) -> None:
    if not isinstance(value, torch.Tensor):
        view.fill_(value)
    elif view.dtype.itemsize == 1:
        view.view(torch.uint8).copy_(value.contiguous().view(torch.uint8))
    else:
        view.copy_(value)


def _check_options(g: dict) -> None:
    lr, (beta1, beta2) = g["lr"], g["betas"]
    if isinstance(lr, torch.Tensor):
        if lr.numel() != 1 or lr.dtype != torch.float32:
            raise ValueError(f"lr as a tensor must be one float32 element, got {tuple(lr.shape)} {lr.dtype}")
    elif not (lr >= 0 and math.isfinite(lr)):
        raise ValueError(f"lr must be 0 or above, got {lr}")
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
        raise ValueError(f"betas must be from 0 to below 1, got {g['betas']}")
    if not g["eps"] >= 0 or not g["weight_decay"] >= 0:
        raise ValueError(f"eps and weight_decay must be 0 or above, got {g['eps']} and {g['weight_decay']}")
    if g["state_bits"] not in (32, 8):
        raise ValueError(f"state_bits must be 32 or 8, got {g['state_bits']}")
    if not (isinstance(g["seed"], int) and 0 <= g["seed"] < 1 << 32):
        raise ValueError(f"seed must be an integer of 32 bits, got {g['seed']}")
    for name in ("amsgrad", "maximize"):
        if g.get(name):
            raise ValueError(f"{name} is not offered")


def _check_state(state: dict | None, p: torch.Tensor, bits: int) -> None:
    if state is None:
        return
    kinds = _kinds(bits)
    if set(state) != {"step", *kinds}:
        raise ValueError(f"a state in {bits} bits holds {sorted(('step', *kinds))}, got {sorted(state)}")
    for name, (dtype, per) in kinds.items():
        shape = tuple(p.shape) if per == 1 else (-(-p.numel() // per),)
        t = state[name]
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != shape:
            got = f"{t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else type(t).__name__
            raise ValueError(f"{name} must be {dtype} {shape}, got {got}")
