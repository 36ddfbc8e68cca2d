"""Plain PyTorch forms of the optimizer ops (:mod:`aggregathor_amd.ops.adamw`):
the CPU path, and what the HIP kernels are compared with.

States are computed in the kernels' order, one rounding an operation, so that
they come out the same bit by bit.
"""

import bisect

import torch

GROUP = 32
_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def grad_norm(grads):
    for g in grads:
        if g.layout != torch.strided or g.device != grads[0].device:
            raise RuntimeError(
                "grad_norm: expected dense tensors on one device")
        if g.dtype not in _TYPES:
            raise RuntimeError("grad_norm: expected fp32, bf16 or fp16, got "
                               f"{g.dtype}")
        if g.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("grad_norm: has no gradient of its own; detach "
                               "the tensors or call it under torch.no_grad()")
    return torch.stack([g.double().square().sum()
                        for g in grads]).sum().sqrt().float()


# ---------------------------------------------------------------------------- #
# 8-bit states


def _groups(n):
    return -(-n // GROUP)


def _flat(t):
    """A dense tensor's elements in the order of its memory."""
    return t.detach().as_strided((t.numel(),), (1,))


def _grouped(x):
    """[n] -> [groups, GROUP], zeros behind the end."""
    n = x.numel()
    return torch.nn.functional.pad(x, (0, _groups(n) * GROUP - n)).view(
        -1, GROUP)


def _exponents(codes, dtype=torch.uint8):
    return codes.to(dtype).view(torch.float8_e8m0fnu)


def state8(param):
    n = param.numel()
    out = []
    for least in (7, 56):  # the exponents that a step gives a group of zeros
        out += [torch.zeros_like(param, dtype=torch.float8_e4m3fn,
                                 requires_grad=False),
                _exponents(torch.full((_groups(n),), least,
                                      device=param.device))]
    return tuple(out)


def values8(codes, scales):
    if codes.dtype != torch.float8_e4m3fn or not _dense(codes) or \
            scales.dtype != torch.float8_e8m0fnu or \
            scales.shape != (_groups(codes.numel()),):
        raise RuntimeError("adamw: expected dense e4m3 codes and an e8m0 scale "
                           f"for every {GROUP} of them")
    out = torch.empty_like(codes, dtype=torch.float32)
    n = codes.numel()
    scaled = _grouped(_flat(codes).float()) * scales.float()[:, None]
    _flat(out).copy_(scaled.view(-1)[:n])
    return out


def exponents_of(top, root):
    """Biased exponents of the groups' scales. ``top``: the largest finite
    ``|m|``, or v where ``root``, of each group."""
    field = top.view(torch.int32) >> 23
    return (((field - 127) >> 1) + 120 if root
            else (field - 7).clamp(min=7))


def _largest(x):
    x = _grouped(x).abs()
    return torch.where(x.isfinite(), x, torch.zeros_like(x)).amax(1)


def round_by_chance(x, exponents, chance, least):
    """Codes of x, ``floor(|x| / scale / quantum + chance / 2**16)`` quanta: up
    with that probability (a constant 2**15 rounds to nearest)."""
    n = x.numel()
    inv = torch.exp2(127. - exponents.float())
    y = (_grouped(x.abs()) * inv[:, None]).view(-1)[:n]
    # The chance goes right below the last bit that stays; below 2^-6, where
    # the quantum stays 2^-9, as if y had 2^-6 to it.
    low = torch.where(y < 2. ** -6, 2. ** -6, 0.)
    bits = ((y + low).view(torch.int32) + (chance.int() << 4)) & -0x100000
    z = bits.view(torch.float32) - low
    z = torch.where(y > 0, z.clamp(min=least * 2. ** -9), z)
    z = torch.copysign(z, x)
    z = torch.where(y.isfinite(), z, torch.full_like(z, float("nan")))
    return z.to(torch.float8_e4m3fn)


def nearest8(x, root):
    """``(codes, scales)`` that stand for x, laid out like it, to nearest."""
    flat = _flat(x.float())
    top = _largest(flat * flat if root else flat)
    exponents = exponents_of(top, root)
    half = torch.full_like(flat, 2. ** 15)
    codes = torch.empty_like(x, dtype=torch.float8_e4m3fn)
    _flat(codes).copy_(round_by_chance(flat, exponents, half,
                                       1. if root else 0.))
    return codes, _exponents(exponents)


def _mix(x):
    x = x ^ (x >> 16)
    x = x * 0x9E3779B1 & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = x * 0x85EBCA77 & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(seed, tensor, step, n, device, begin=0):
    """32 random bits for each of the elements [begin, begin + n)."""
    key = _mix(torch.tensor((seed + 0x9E3779B9 * (tensor + 1)) & 0xFFFFFFFF))
    key = int(_mix(key + step & 0xFFFFFFFF))
    at = torch.arange(begin, begin + n, device=device)
    return _mix((at & 0xFFFFFFFF) ^ (key + 0x9E3779B9 * (at >> 32)
                                     & 0xFFFFFFFF))


# ---------------------------------------------------------------------------- #
# Plan


def _same_layout(a, b):
    return a.shape == b.shape and (a.numel() < 2 or all(
        s == 1 or x == y for s, x, y in zip(a.shape, a.stride(), b.stride())))


def _dense(t):
    expected = 1
    for stride, size in sorted((st, si) for st, si in
                               zip(t.stride(), t.shape) if si != 1):
        if stride != expected:
            return t.numel() == 0
        expected *= size
    return True


def _range(t):
    if t.numel() == 0:
        return None
    last = sum((si - 1) * st for si, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _check(ok, message):
    if not ok:
        raise RuntimeError("adamw: " + message)


class Plan:
    """The kernels' plan, in plain PyTorch."""

    def __init__(self, bits, params, m, ms, r, rs, steps, seed, places):
        self.bits, self.seed, self.steps = bits, seed, steps
        self.places = places
        self.params, self.m, self.ms, self.r, self.rs = params, m, ms, r, rs
        self._lay_out()

    def _memory(self):
        """Where the plan's tensors lie, and how. (What they were laid out
        with is out of date once one has got other memory: `param.data = ...`,
        or a module moved.)"""
        return [(t.data_ptr(), t.shape, t.stride(), t.dtype, t.device)
                for t in (self.steps, *self.params, *self.m, *self.ms,
                          *self.r, *self.rs)]

    def _lay_out(self):
        bits, steps = self.bits, self.steps
        params, m, ms, r, rs = self.params, self.m, self.ms, self.r, self.rs
        count, device = len(params), params[0].device
        _check(len(m) == len(r) == count and
               (bits == 32 or len(ms) == len(rs) == count),
               "as many states as parameters are needed")
        _check(len(self.places) == count,
               "as many places as parameters are needed")
        _check(steps.device == device and steps.shape == (count,)
               and steps.is_contiguous() and steps.dtype == torch.int32,
               "steps is a contiguous int32 tensor of one count for each "
               "parameter, on their device")
        kind = torch.float8_e4m3fn if bits == 8 else torch.float32
        written = [steps]
        for i, p in enumerate(params):
            _check(p.dtype in _TYPES, f"parameter {i}: expected fp32, bf16 or "
                   f"fp16, got {p.dtype}")
            _check(p.layout == torch.strided, "expected dense parameters")
            _check(p.device == device,
                   "the parameters of a plan are on one device")
            _check(_dense(p), f"parameter {i} of shape {tuple(p.shape)} and "
                   f"strides {p.stride()} does not fill its memory")
            _check(not p.is_neg(), f"parameter {i} is a view that negates")
            for name, s in (("exp_avg", m[i]), (
                    "exp_avg_root" if bits == 8 else "exp_avg_sq", r[i])):
                _check(s.dtype == kind,
                       f"{name} {i} is {s.dtype}, expected {kind}")
                _check(s.device == device, f"{name} {i} is on {s.device}, its "
                       f"parameter on {device}")
                _check(not s.is_neg(), f"{name} {i} is a view that negates")
                _check(_same_layout(s, p), f"{name} {i} has another shape or "
                       "other strides than its parameter")
            written += [p, m[i], r[i]]
            if bits == 8:
                for s in (ms[i], rs[i]):
                    _check(s.dtype == torch.float8_e8m0fnu
                           and s.device == device and s.is_contiguous()
                           and s.shape == (_groups(p.numel()),),
                           f"the scales of state {i} are a contiguous e8m0 "
                           f"tensor of {_groups(p.numel())} elements on its "
                           "parameter's device")
                    written.append(s)
        ranges = sorted(x for x in map(_range, written) if x)
        _check(all(a[1] <= b[0] for a, b in zip(ranges, ranges[1:])),
               "parameters, states and steps share memory")
        self.ranges, self.ends = ranges, [hi for _, hi in ranges]
        self.memory = self._memory()

    def _check_apart(self, t, what):
        r = _range(t)
        # The first range that ends behind the tensor's begin.
        i = 0 if r is None else bisect.bisect_right(self.ends, r[0])
        _check(r is None or i == len(self.ranges)
               or r[1] <= self.ranges[i][0],
               f"{what} shares memory with a parameter or state")

    @torch.no_grad()
    def step(self, grads, lr, beta1, beta2, eps, weight_decay, norm, max_norm):
        grads = list(grads)
        device = self.params[0].device
        _check(len(grads) == len(self.params), f"{len(self.params)} "
               f"parameters, but {len(grads)} gradients")
        if self._memory() != self.memory:
            self._lay_out()
        clip = None
        if norm is not None:
            _check(norm.device == device and norm.numel() == 1
                   and norm.dtype == torch.float32 and not norm.is_neg(),
                   "norm is one fp32 number on the parameters' device, and no "
                   "view that negates")
            self._check_apart(norm, "norm")
            clip = torch.where(norm <= max_norm, torch.ones_like(norm),
                               max_norm / norm).reshape(())
        for i, (g, p) in enumerate(zip(grads, self.params)):
            if g is None:
                continue
            _check(g.layout == torch.strided, f"gradient {i} is not dense")
            _check(g.device == device, f"gradient {i} is on {g.device}, its "
                   f"parameter on {device}")
            _check(g.shape == p.shape, f"gradient {i} has the shape "
                   f"{tuple(g.shape)}, its parameter {tuple(p.shape)}")
            _check(g.dtype in _TYPES and
                   (g.dtype == p.dtype or p.dtype == torch.float32),
                   f"gradient {i} is {g.dtype}, its parameter {p.dtype} (the "
                   "same type, or fp32 parameters)")
            self._check_apart(g, "gradient")
        for i, (g, p) in enumerate(zip(grads, self.params)):
            if g is not None:
                self._step_one(i, g, p, lr, beta1, beta2, eps, weight_decay,
                               clip)

    def _step_one(self, i, g, p, lr, beta1, beta2, eps, weight_decay, clip):
        if not _same_layout(g, p):
            g = torch.empty_like(p, dtype=g.dtype).copy_(g)
        g = _flat(g.resolve_neg()).float()
        if clip is not None:
            g = g * clip
        self.steps[i] += 1
        t = self.steps[i].double()
        rate = (lr / (1 - beta1 ** t)).float()
        unbias = (1 / (1 - beta2 ** t).sqrt()).float()
        ms, rs = _flat(self.m[i]), _flat(self.r[i])
        if self.bits == 32:
            m, v = ms, rs
        else:
            m = _flat(values8(ms, self.ms[i]))
            v = _flat(values8(rs, self.rs[i])).square()
        m = m * beta1 + g * (1 - beta1)
        v = v * beta2 + g * g * (1 - beta2)
        # Through 64 bits: the CPU's vector library is off in the last one.
        root = v.double().sqrt().float()
        moved = (_flat(p).float() * (1 - lr * weight_decay)
                 - rate * (m / (root * unbias + eps)))
        # copy_ through the parameter, so that autograd sees the change.
        p.as_strided((p.numel(),), (1,)).copy_(moved)
        if self.bits == 32:
            ms.copy_(m)
            rs.copy_(v)
            return
        bits = random_bits(self.seed, self.places[i], int(self.steps[i]),
                           p.numel(), p.device)
        for codes, scales, x, of, root_, chance in (
                (ms, self.ms[i], m, m, False, bits & 0xFFFF),
                (rs, self.rs[i], root, v, True, bits >> 16)):
            exponents = exponents_of(_largest(of), root_)
            scales.copy_(_exponents(exponents))
            codes.copy_(round_by_chance(x, exponents, chance.float(),
                                        1. if root_ else 0.))
