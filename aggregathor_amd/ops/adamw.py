"""Optimizer ops: the norm over many tensors, and the AdamW step over many
tensors with states in 32 or in 8 bits.

With ``g`` the gradient, ``t`` the tensor's number of steps and
``s = 1 if norm <= max_norm else max_norm / norm`` (1 without a norm)::

    m = beta1 * m + (1 - beta1) * s * g
    v = beta2 * v + (1 - beta2) * (s * g)**2
    p = p * (1 - lr * weight_decay)
        - lr / (1 - beta1**t) * m / (sqrt(v) / sqrt(1 - beta2**t) + eps)

A plan holds the tensors of a training run (parameters, states, step counts)
the way an optimizer does, checked and laid out once; each call of
:func:`adamw_step` brings the gradients. Laying it out takes longer than a step
(0.3 ms for ResNet-50 on a GPU): every tensor is checked, and a table of 64
bytes for each 1024 elements (2048 of large 8-bit states) is sent to the device,
which is waited for. A step whose tensors have other memory than in the last one
(``param.data = ...``) does it again. :class:`aggregathor_amd.optim.AdamW` is the
optimizer on top.

Tensors are dense in any order of their dimensions (contiguous, channels
last, ...), with any number of elements, zero among them. Parameters are fp32,
bf16 or fp16 with gradients of their type, or fp32 with bf16 or fp16 gradients.
All arithmetic is in fp32. Parameters of 16 bits are rounded to nearest at the
end of each step, so what a step moves them by less than half their last bit is
lost; fp32 parameters under autocast have no such loss.

States of 8 bits (:func:`adamw8_plan`) take 2.06 bytes an element instead of 8:
``m`` and ``r = sqrt(v)`` are e4m3 codes, and every 32 elements that follow
each other in the tensor's memory share a power of two. Codes are rounded up or
down by chance, without bias, from a hash of the plan's seed, the tensor's place
in it, its step count and the element's place: the same inputs give the same
bits, on every rank. The step itself uses ``m`` and ``v`` before they are
rounded. A group may hold 17 binades: what is further below its largest value
becomes zero or the least code by chance (never zero for ``r``).
NaN and infinities spread as the formulas say; an 8-bit state stores either as
NaN, without harm to the other elements of its group.

GPU tensors take the gfx950 kernels (``csrc/adamw_kernels.hip``), CPU tensors
the plain PyTorch forms of :mod:`aggregathor_amd.ops.adamw_reference`.
"""

import math

import torch

from . import _load_extension, _want_hip
from . import adamw_reference as reference

#: Elements that share a scale in an 8-bit state.
GROUP = reference.GROUP


def _ext(tensor):
    """The HIP extension for a GPU tensor, None for the plain forms."""
    return _load_extension() if _want_hip(tensor) else None


def grad_norm(grads):
    """L2 norm over all elements of a tensor, or of all tensors of a list, as one
    fp32 number on their device (nothing waits for it). Squares are summed in 64
    bits, in an order that the tensors' sizes and places in memory alone set: the
    same tensors have the same norm every time, equal ones elsewhere may have
    another last bit (those that lie back to back are read as one). It is not
    differentiable: tensors that need a gradient are refused, but under
    ``torch.no_grad()``."""
    if isinstance(grads, torch.Tensor):
        grads = (grads,)
    elif not isinstance(grads, (list, tuple)):
        grads = list(grads)
    if not grads:
        raise RuntimeError("grad_norm: expected a tensor")
    ext = _ext(grads[0])
    return (reference if ext is None else ext).grad_norm(grads)


def _plan(bits, params, m, ms, r, rs, steps, seed, places=None):
    params = list(params)
    if not params:
        raise RuntimeError("adamw: a plan needs a parameter")
    ext = _ext(params[0])
    make = reference.Plan if ext is None else ext.AdamWPlan
    places = range(len(params)) if places is None else places
    return make(bits, params, list(m), list(ms), list(r), list(rs), steps,
                int(seed) & 0xFFFFFFFF, [int(i) & 0xFFFFFFFF for i in places])


def adamw_plan(params, exp_avgs, exp_avg_sqs, steps):
    """A plan over 32-bit states.

    Args:
      params:      the parameter tensors (all on one device)
      exp_avgs:    m of each, fp32, shaped and strided like it
      exp_avg_sqs: v of each, likewise
      steps:       int32 tensor on their device, the number of steps that each
                   parameter has had
    """
    return _plan(32, params, exp_avgs, (), exp_avg_sqs, (), steps, 0)


def adamw8_plan(params, exp_avgs, exp_avg_scales, exp_avg_roots,
                exp_avg_root_scales, steps, seed=0, places=None):
    """A plan over 8-bit states (made by :func:`adamw8_state`).

    Args:
      params:              the parameter tensors (all on one device)
      exp_avgs:            float8_e4m3fn codes of m, shaped and strided like it
      exp_avg_scales:      float8_e8m0fnu, one for 32 elements
      exp_avg_roots:       codes of sqrt(v)
      exp_avg_root_scales: their scales
      steps:               int32 tensor, as of :func:`adamw_plan`
      seed:                of the rounding (its low 32 bits)
      places:              of each parameter, the number that stands for it in
                           the rounding (None: 0, 1, ...); with its own it is
                           rounded alike in any plan
    """
    return _plan(8, params, exp_avgs, exp_avg_scales, exp_avg_roots,
                 exp_avg_root_scales, steps, seed, places)


def adamw8_state(param):
    """Zero states of 8 bits for a parameter: ``(exp_avg, exp_avg_scale,
    exp_avg_root, exp_avg_root_scale)``."""
    return reference.state8(param)


def adamw8_values(codes, scales):
    """The values (fp32, laid out like ``codes``) that an 8-bit state stands
    for: m of an ``exp_avg``, sqrt(v) of an ``exp_avg_root``."""
    return reference.values8(codes, scales)


def out_of_range(lr, beta1, beta2, eps, weight_decay, max_norm=None):
    """What is wrong with the settings of a step, None where nothing is."""
    for name, value, ok in (
            ("lr", lr, 0. <= lr < math.inf),
            ("beta1", beta1, 0. <= beta1 < 1.),
            ("beta2", beta2, 0. <= beta2 < 1.),
            # Normal numbers, also behind a division: the kernels' reciprocal
            # takes others for zero.
            ("eps", eps, 1.2e-38 <= eps <= 1e30),
            ("weight_decay", weight_decay, 0. <= weight_decay < math.inf),
            ("max_norm", max_norm,
             max_norm is None or 1.2e-38 <= max_norm < 3e38)):
        if not ok:
            return f"{name} = {value} is out of range"
    return None


def adamw_step(plan, grads, lr, beta1=0.9, beta2=0.999, eps=1e-8,
               weight_decay=0.01, norm=None, max_norm=None):
    """One AdamW step over all tensors of a plan, in place.

    Args:
      plan:     of :func:`adamw_plan` or :func:`adamw8_plan`
      grads:    the gradient of each parameter, or None: that parameter, its
                state and its step count stay as they are. A gradient whose
                strides are not its parameter's is copied first.
      norm:     one fp32 number on the device (:func:`grad_norm`); gradients
                are scaled by max_norm / norm where it exceeds
      max_norm: that limit. A NaN norm makes every parameter NaN, an infinite
                one scales finite gradients to zero.

    Launches go to the current stream; inside a graph capture they are recorded
    (step counts live on the device, so every replay is a step of its own).
    Work on a plan from two streams has to be ordered by the caller, as for any
    tensors that are updated in place.
    """
    refusal = out_of_range(lr, beta1, beta2, eps, weight_decay, max_norm)
    if refusal:
        raise RuntimeError("adamw: " + refusal)
    if (norm is None) != (max_norm is None):
        raise RuntimeError("adamw: norm and max_norm belong together")
    if max_norm is None:
        max_norm = 1.
    if not isinstance(grads, (list, tuple)):
        grads = list(grads)
    plan.step(grads, lr, beta1, beta2, eps, weight_decay, norm, max_norm)
