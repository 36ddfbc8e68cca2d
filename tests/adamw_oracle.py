"""The AdamW step in 64 bits, with the bounds that fp32 arithmetic keeps to.

With u = 2^-24, half a step of fp32 relative to the value, and each constant and
each operation off by at most u (the clip factor by 2u: the norm's own rounding
and the division), to first order:

  s g         3u
  m           beta1 m: 2u, (1 - beta1) s g: 5u, the sum: u
              -> 6u M with M = beta1 |m| + (1 - beta1) |s g|
  v           beta2 v: 2u, (1 - beta2) (s g)^2: 9u, the sum: u -> 10u v
  root        half of v's, and u -> 6u
  denominator root unbias: 8u, eps: u, the sum: u -> 9u
  step        6u M / m, 9u, the division u, the rate u, the product u
              -> at most 18u rate M / denominator
  p           keep p: 2u |p|, the step, the sum: u |p'|

A square root, a division or a reciprocal that is off by a unit in the last
place rather than half adds 2u each where it enters. The bounds below leave room
for that, and for what is of second order.
"""

import torch

U = 2. ** -24
TINY = 2. ** -149


def clip_factor(grads, max_norm):
    """(norm, factor) in 64 bits."""
    norm = sum(float(g.double().square().sum()) for g in grads
               if g is not None) ** .5
    return norm, 1. if norm <= max_norm else max_norm / norm


def step(p, g, m, v, t, lr, beta1, beta2, eps, weight_decay, s=1.):
    """One step of one tensor: ((p, m, v), (bounds)), t the count after it."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * s
    M = beta1 * m.abs() + (1 - beta1) * g.abs()
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    rate = lr / (1 - beta1 ** t)
    denominator = v.sqrt() / (1 - beta2 ** t) ** .5 + eps
    moved = p * (1 - lr * weight_decay) - rate * m / denominator
    bounds = (3 * U * p.abs() + 2 * U * moved.abs()
              + 26 * U * rate * M / denominator + TINY,
              8 * U * M + 4 * TINY, 12 * U * v + 4 * TINY)
    return (moved, m, v), bounds


def rounded(bound, value, dtype):
    """The bound of a value that is rounded once more, to `dtype`."""
    if dtype == torch.float32:
        return bound
    info = torch.finfo(dtype)
    return bound + info.eps / 2 * (value.abs() + bound) + \
        info.smallest_normal * info.eps / 2


def check(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.cpu()
    off = (got - want).abs() - bound.cpu()
    assert bool((off <= 0).all()), \
        f"{what}: {float(off.max()):.3g} beyond its bound"


def check8(codes, scales, values, x, root, what):
    """8-bit states against x, what they stand for before rounding: within one
    quantum of it (an eighth of the power of two below it, or the format's
    least step), and every group's scale the least that holds its largest."""
    x = x.double().cpu().reshape(-1)
    values = values.detach().double().cpu().reshape(-1)
    scales = scales.float().double().cpu().repeat_interleave(32)[:x.numel()]
    near = x.abs() * (1 + 16 * U)
    quantum = torch.maximum(near / 8, scales * 2. ** -9)
    off = (values - x).abs() - quantum * (1 + 16 * U)
    # A root may be raised to the least code above zero: within that quantum.
    assert bool((off <= 0).all()), f"{what}: {float(off.max()):.3g} too far"
    assert bool((near / scales < 256.001).all()), f"{what}: scale too small"
    if root:
        assert bool(((values > 0) == (x > 0)).all()), f"{what}: zero roots"
