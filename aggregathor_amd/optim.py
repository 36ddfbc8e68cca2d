"""AdamW over the framework's optimizer kernels (:mod:`aggregathor_amd.ops`).

One launch updates all parameters of a group (one for each 448 of them); step
counts, clipping and the rounding's random bits live on the device, so a step
waits for nothing and can be captured into a graph (a captured
``torch.optim.Adam`` needs ``capturable=True`` for that). States take 8 bytes an
element, or 2.06 with ``state_bits=8``.

The result is a function of parameters, gradients and states alone, bit by bit:
ranks that hold the same aggregated gradient keep the same parameters. With
clipping, the gradients have to lie alike in memory for that (as views into one
flat buffer do, which is what the engine has): the norm adds up tensors that lie
back to back as one, so that its last bit may be another for the same gradients
in separate memory.
"""

from itertools import chain, starmap, zip_longest
from operator import is_

import torch

from . import ops, tools
from .ops import adamw_reference as reference
from .ops.adamw import out_of_range

_STATES = {32: ("exp_avg", "exp_avg_sq"),
           8: ("exp_avg", "exp_avg_scale", "exp_avg_root",
               "exp_avg_root_scale")}


class _Held:
    """A plan, and the parameters and states that it is over."""

    def __init__(self, group, params, plan, tensors):
        self.group, self.params, self.plan = group, params, plan
        self._tensors = tensors  # of each parameter's state, by name

    def holds(self, states):
        """Whether the states are still those."""
        return all(states.get(p, {}).get(name) is tensor
                   for p, tensors in zip(self.params, self._tensors)
                   for name, tensor in tensors.items())


class AdamW(torch.optim.Optimizer):
    """AdamW (Adam with decoupled weight decay).

    Args:
      params:        parameters or parameter groups
      lr, betas, eps, weight_decay: as in ``torch.optim.AdamW`` (per group)
      state_bits:    32 or 8, the width of the states (per group)
      max_norm:      clip the gradient of all groups together to this L2 norm
                     (None: no clipping; parameters on one device only)
      rounding_seed: of the 8-bit states' rounding

    A parameter without a gradient is left out of the step, its step count too;
    it has no state before it first has a gradient.
    Each parameter's ``state`` holds ``step`` and the state tensors; they may be
    changed in place, replaced, or cleared (the next step starts from zero
    there). :meth:`load_state_dict` replaces them; it also takes the state of a
    ``torch.optim.AdamW``, or of an ``Adam`` without weight decay (32 bits).

    A captured step goes on with the parameters and states that it was captured
    with: where these are replaced, it has to be captured again.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=1e-2, state_bits=32, max_norm=None,
                 rounding_seed=0):
        self.max_norm = max_norm
        self.rounding_seed = rounding_seed
        self._plans, self._laid_out = [], False
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps,
                                      weight_decay=weight_decay,
                                      state_bits=state_bits))

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            self._check_bits(group)
            refusal = self._refusal(group)
            if refusal:
                raise tools.UserException("adamw: " + refusal)
        except Exception:
            self.param_groups.pop()
            raise
        self._laid_out = False

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans, self._laid_out = [], False

    def __getstate__(self):
        # Plans are laid out anew where the optimizer is copied to.
        return dict(super().__getstate__(), max_norm=self.max_norm,
                    rounding_seed=self.rounding_seed)

    def _refusal(self, group):
        """What is wrong with a group's settings."""
        return out_of_range(float(group["lr"]), *group["betas"], group["eps"],
                            group["weight_decay"], self.max_norm)

    @staticmethod
    def _check_bits(group):
        if group["state_bits"] not in _STATES:
            raise tools.UserException("adamw: states have 32 or 8 bits, not "
                                      f"{group['state_bits']!r}")

    # ------------------------------------------------------------------ #

    def _lay_out(self):
        """Plans over the parameters that have a gradient or a state, where
        there is none over their states: one for each group (and each device)
        and each time that some of its parameters are the first to have one.
        What a plan holds stays where it is, also for a captured step."""
        self._laid_out = False
        self._plans = [plan for plan in self._plans if plan.holds(self.state)]
        held = {p for plan in self._plans for p in plan.params}
        waiting = []
        for index, group in enumerate(self.param_groups):
            by_device, places = {}, {}
            for p in group["params"]:
                # Its number among the group's on its device, whether or not
                # the others are there.
                place = places[p.device] = places.get(p.device, -1) + 1
                if p in held:
                    continue
                if p.grad is None and not self.state.get(p):
                    waiting.append(p)
                else:
                    by_device.setdefault(p.device, []).append((place, p))
            for device, params in by_device.items():
                if torch.cuda.is_available() and \
                        torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(
                        "adamw: run a step before the capture, so that the "
                        "states and plans are there")
                self._check_bits(group)
                self._plans.append(self._plan(group, index, device,
                                              *zip(*params)))
        there = [p for plan in self._plans for p in plan.params]
        held = set(there)
        self._in_order = all(map(is_, there, (
            p for group in self.param_groups for p in group["params"]
            if p in held)))
        self._waiting = waiting
        self._seen = list(self._all_states())
        self._laid_out = True

    def _all_states(self):
        return chain.from_iterable(map(dict.values, self.state.values()))

    def _states_kept(self):
        """Whether all states are what they were (a caller may have cleared or
        replaced some). Without a lookup by parameter, which hashes it in
        Python: 161 parameters took 59 us so, and take 17."""
        return all(starmap(is_, zip_longest(self._all_states(), self._seen,
                                            fillvalue=self)))

    def _plan(self, group, index, device, places, params):
        bits = group["state_bits"]
        steps = torch.zeros(len(params), dtype=torch.int32, device=device)
        columns = [[] for _ in _STATES[bits]]
        for i, p in enumerate(params):
            state = self.state[p]
            if "step" in state:
                missing = set(_STATES[bits]) - set(state)
                if missing:
                    raise RuntimeError("adamw: a state lacks " + ", ".join(
                        sorted(missing)))
                steps[i] = state["step"]
            else:
                fresh = (ops.adamw8_state(p) if bits == 8 else
                         [torch.zeros_like(p, dtype=torch.float32,
                                           requires_grad=False)
                          for _ in range(2)])
                state.update(zip(_STATES[bits], fresh))
            state["step"] = steps[i]  # a view: the plan counts there
            for column, name in zip(columns, _STATES[bits]):
                column.append(state[name])
        if bits == 8:
            plan = ops.adamw8_plan(params, *columns, steps,
                                   seed=self.rounding_seed + index,
                                   places=places)
        else:
            plan = ops.adamw_plan(params, *columns, steps)
        names = ("step", *_STATES[bits])
        return _Held(group, params, plan,
                     [{name: self.state[p][name] for name in names}
                      for p in params])

    @torch.no_grad()
    def step(self, closure=None):
        """One step over all parameters that have a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if not self._laid_out or not self._states_kept() or any(
                p.grad is not None for p in self._waiting):
            self._lay_out()
        grads = [[p.grad for p in held.params] for held in self._plans]
        norm = None
        if self.max_norm is not None:
            # In the order of the parameters, which the sum's depends on.
            present = [g for part in (grads if self._in_order else (
                [p.grad for p in group["params"]]
                for group in self.param_groups)) for g in part
                       if g is not None]
            if not present:
                return loss
            norm = ops.grad_norm(present)
        for held, part in zip(self._plans, grads):
            group = held.group
            beta1, beta2 = group["betas"]
            ops.adamw_step(held.plan, part, lr=float(group["lr"]), beta1=beta1,
                           beta2=beta2, eps=group["eps"],
                           weight_decay=group["weight_decay"], norm=norm,
                           max_norm=self.max_norm)
        return loss

    # ------------------------------------------------------------------ #

    def load_state_dict(self, state_dict):
        """Load what :meth:`state_dict` gave. (The base class would cast every
        state to its parameter's type: it gets none to cast.)"""
        states = {}

        def take(_, given):  # behind the caller's hooks, which may change it
            groups, found = self._readable(given)
            states.update(found)
            return {"state": {}, "param_groups": groups}

        def keep(_):  # ahead of the caller's hooks, which may look at it
            self.state.update(states)
            self._plans, self._laid_out = [], False

        hooks = (self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(keep, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _readable(self, state_dict):
        """The groups and states of a state dict, where the optimizer can go on
        with them."""
        groups = []
        for given in state_dict["param_groups"]:
            group = {**self.defaults, **given}
            if state_dict["state"] and "state_bits" not in given:
                group["state_bits"] = 32  # torch's own
            self._check_bits(group)
            refusal = self._refusal(group)
            if refusal:
                raise ValueError("loaded state dict: " + refusal)
            for other in ("amsgrad", "maximize"):
                if group.get(other):
                    raise ValueError(f"loaded state dict is of a step with "
                                     f"{other}, which this optimizer has not")
            # torch's Adam adds its decay to the gradient (and says so; what is
            # no Adam at all has no betas).
            if given.get("weight_decay") and "state_bits" not in given and \
                    not given.get("decoupled_weight_decay", "betas" in given):
                raise ValueError("loaded state dict is of a step whose weight "
                                 "decay goes through the gradient; here it is "
                                 "decoupled")
            groups.append(group)
        saved = [i for group in groups for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        bits = [group["state_bits"] for group in groups
                for _ in group["params"]]
        if len(saved) != len(params):
            raise ValueError("loaded state dict has another number of "
                             "parameters than the optimizer")
        states = {p: self._loaded(state_dict["state"][i], p, b)
                  for i, p, b in zip(saved, params, bits)
                  if state_dict["state"].get(i)}
        return groups, states

    @staticmethod
    def _loaded(state, p, bits):
        missing = {"step", *_STATES[bits]} - set(state)
        if missing:
            raise ValueError("loaded state dict lacks " + ", ".join(
                sorted(missing)) + f" of a state of {bits} bits")
        # A copy: the state may be another optimizer's, which goes on.
        out = {"step": torch.as_tensor(state["step"]).to(torch.int32,
                                                         copy=True)}
        names = _STATES[32] if bits == 32 else ("exp_avg", "exp_avg_root")
        for name in names:
            if state[name].shape != p.shape:
                raise ValueError(f"loaded {name} has the shape "
                                 f"{tuple(state[name].shape)}, its parameter "
                                 f"{tuple(p.shape)}")
        if bits == 32:
            for name in names:
                out[name] = torch.empty_like(
                    p, dtype=torch.float32, requires_grad=False).copy_(
                        state[name])
            return out
        for name in names:
            codes = state[name]
            scales = state[name + "_scale"]
            if codes.dtype != torch.float8_e4m3fn or \
                    scales.dtype != torch.float8_e8m0fnu:
                raise ValueError(f"loaded {name} is no 8-bit state")
            if scales.shape != (-(-codes.numel() // reference.GROUP),):
                raise ValueError(f"loaded {name}_scale has the shape "
                                 f"{tuple(scales.shape)}, not one element for "
                                 f"{reference.GROUP} of {name}")
            if reference._same_layout(codes, p):
                codes, scales = codes.clone(), scales.clone()
            else:
                # Groups follow the memory: another order of the dimensions
                # (contiguous on the CPU, channels last on a GPU) has others.
                values = torch.empty_like(
                    p, dtype=torch.float32, requires_grad=False,
                    device=codes.device).copy_(
                        reference.values8(codes, scales))
                codes, scales = reference.nearest8(
                    values, root=name == "exp_avg_root")
            out[name] = codes.to(p.device)
            out[name + "_scale"] = scales.to(p.device)
        return out
