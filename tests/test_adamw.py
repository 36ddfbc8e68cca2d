"""Optimizer ops and AdamW on the CPU: the plain forms against 64 bits, the
8-bit states' rounding, refusals, checkpoints, the engine."""

import copy
import io
import math
import os
import pathlib
import re
import shutil
import subprocess
import sys

import pytest
import torch

import adamw_oracle as oracle
from aggregathor_amd import ops
from aggregathor_amd.graph import Engine, build_optimizer
from aggregathor_amd.ops import adamw_reference as R
from aggregathor_amd.ops import build as ops_build
from aggregathor_amd.optim import AdamW
from aggregathor_amd.parallel import WorkerGroup
from aggregathor_amd import experiments, tools

SIZES = [1, 3, 31, 32, 33, 100, 257, 0]


def _tensors(sizes, dtype=torch.float32, seed=0, scale=1.):
    gen = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(n, generator=gen)).to(dtype) for n in sizes]


def _state32(params, seed=1):
    m = [0.1 * t for t in _tensors([p.numel() for p in params], seed=seed)]
    v = [t.square() * 0.02 for t in _tensors([p.numel() for p in params],
                                             seed=seed + 1)]
    return m, v


def _state8(params, seed=1):
    m, v = _state32(params, seed)
    out = [R.nearest8(x, False) + R.nearest8(y.sqrt(), True)
           for x, y in zip(m, v)]
    return [list(column) for column in zip(*out)]


def _steps(*counts):
    return torch.tensor(counts, dtype=torch.int32)


# ---------------------------------------------------------------------------- #
# Norm


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
def test_grad_norm(dtype):
    grads = _tensors(SIZES, dtype)
    want = sum(float(g.double().square().sum()) for g in grads) ** .5
    got = ops.grad_norm(grads)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= 2 * oracle.U * want


def test_grad_norm_extremes():
    assert float(ops.grad_norm([torch.zeros(5), torch.zeros(0)])) == 0
    assert float(ops.grad_norm(torch.full((4,), 1e30))) == pytest.approx(2e30)
    assert float(ops.grad_norm(torch.full((4,), 1e-30))) == pytest.approx(
        2e-30)
    assert math.isnan(float(ops.grad_norm([torch.tensor([float("nan"), 1.])])))
    assert math.isinf(float(ops.grad_norm([torch.tensor([-math.inf, 1.])])))


# ---------------------------------------------------------------------------- #
# Step


@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
@pytest.mark.parametrize("p_dtype,g_dtype", [
    (torch.float32, torch.float32), (torch.float32, torch.bfloat16),
    (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_step32_against_64_bits(p_dtype, g_dtype, max_norm):
    params = _tensors(SIZES, p_dtype)
    grads = _tensors(SIZES, g_dtype, seed=5, scale=0.3)
    m, v = _state32(params)
    counts = [0, 1, 7, 100, 5000, 3, 2, 1]
    steps = _steps(*counts)
    hyper = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.1)
    norm, s = (None, 1.) if max_norm is None else oracle.clip_factor(
        grads, max_norm)
    want = [oracle.step(*x, t + 1, **hyper, s=s)
            for *x, t in zip(params, grads, m, v, counts)]
    plan = ops.adamw_plan(params, m, v, steps)
    ops.adamw_step(plan, grads, **hyper, max_norm=max_norm,
                   norm=None if norm is None else ops.grad_norm(grads))
    assert steps.tolist() == [t + 1 for t in counts]
    for i, (values, bounds) in enumerate(want):
        bounds = (oracle.rounded(bounds[0], values[0], p_dtype), *bounds[1:])
        for name, got, x, b in zip("pmv", (params[i], m[i], v[i]), values,
                                   bounds):
            oracle.check(got, x, b, f"{name} of {SIZES[i]}")


def test_step8_against_64_bits():
    params = _tensors(SIZES)
    grads = _tensors(SIZES, seed=5, scale=0.3)
    m, ms, r, rs = _state8(params)
    hyper = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.1)
    values = [(R.values8(a, b), R.values8(c, d).square())
              for a, b, c, d in zip(m, ms, r, rs)]
    want = [oracle.step(p, g, *mv, 4, **hyper)
            for p, g, mv in zip(params, grads, values)]
    ops.adamw_step(ops.adamw8_plan(params, m, ms, r, rs, _steps(*[3] * 8)),
                   grads, **hyper)
    for i, (x, bounds) in enumerate(want):
        oracle.check(params[i], x[0], bounds[0], f"p of {SIZES[i]}")
        oracle.check8(m[i], ms[i], ops.adamw8_values(m[i], ms[i]), x[1],
                      False, f"m of {SIZES[i]}")
        oracle.check8(r[i], rs[i], ops.adamw8_values(r[i], rs[i]),
                      x[2].sqrt(), True, f"r of {SIZES[i]}")


def test_a_missing_gradient_leaves_all_as_it_was():
    params = _tensors([5, 40, 7])
    m, ms, r, rs = _state8(params)
    steps = _steps(4, 4, 4)
    before = copy.deepcopy([params[1], m[1].float(), ms[1].float(),
                            r[1].float(), rs[1].float()])
    ops.adamw_step(ops.adamw8_plan(params, m, ms, r, rs, steps),
                   [torch.ones(5), None, torch.ones(7)], lr=0.1)
    assert steps.tolist() == [5, 4, 5]
    for x, y in zip(before, (params[1], m[1], ms[1], r[1], rs[1])):
        assert torch.equal(x, y.float())


def test_rounding_has_no_bias():
    # Over all 2^16 values of the chance, the mean code is the value itself but
    # for the chance's own grain, 2^-16 of a quantum.
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(32, generator=gen) * torch.logspace(0, -6, 32)
    exponents = R.exponents_of(R._largest(x), False)
    scale = 2. ** (float(exponents) - 127)
    chance = torch.arange(65536.)
    for value in x.tolist():
        one = torch.full((65536,), value)
        # The group's exponent is given, not taken from these copies.
        codes = R.round_by_chance(one, exponents.expand(2048), chance, 0.)
        mean = float(codes.double().mean()) * scale
        quantum = max(2. ** (math.floor(math.log2(abs(value) / scale)) - 3),
                      2. ** -9) * scale
        assert abs(mean - value) <= 2. ** -16 * quantum * 1.0001


def test_values_on_the_grid_stay():
    grid = torch.arange(128, 256, 16.).repeat(4)  # of one group
    codes, scales = R.nearest8(grid, False)
    assert torch.equal(R.values8(codes, scales), grid)
    for chance in (0., 65535.):
        again = R.round_by_chance(grid, scales.view(torch.uint8).int(),
                                  torch.full((32,), chance), 0.)
        assert torch.equal(again.float(), codes.float())


def test_random_bits_look_random():
    bits = R.random_bits(7, 2, 5, 1 << 16, "cpu")
    other = R.random_bits(7, 2, 6, 1 << 16, "cpu")
    half = [(b.double() / 65536 - 0.5) for x in (bits, other)
            for b in (x & 0xFFFF, x >> 16)]
    # A mean of N uniform numbers is off by 1/sqrt(12 N) = 0.0011 (5 of these).
    for h in half:
        assert abs(float(h.mean())) < 0.006
    for i in range(4):
        for j in range(i):
            c = float((half[i] * half[j]).mean() * 12)  # 1/sqrt(N) = 0.004
            assert abs(c) < 0.02
    assert torch.equal(R.random_bits(7, 2, 5, 100, "cpu", begin=200),
                       bits[200:300])


def test_state8_of_extremes():
    inf, nan = math.inf, math.nan
    x = torch.zeros(96)
    x[:6] = torch.tensor([3e38, -3e38, 1e-30, inf, nan, 0.])
    x[32:36] = torch.tensor([1e-45, -1e-40, 1e-38, 0.])
    codes, scales = R.nearest8(x, False)
    back = R.values8(codes, scales)
    assert back[:2].tolist() == pytest.approx([3e38, -3e38], rel=2. ** -4)
    assert back[2] == 0 and back[5] == 0
    assert back[3].isnan() and back[4].isnan()
    # Half a quantum of the least scale, 2^-120 2^-9.
    assert (back[32:36] - x[32:36]).abs().max() <= 2. ** -130 * 1.01
    assert torch.equal(back[64:], torch.zeros(32))


def test_roots_never_become_zero():
    params = [torch.zeros(64)]
    m, ms, r, rs = _state8(params, seed=9)
    grad = torch.full((64,), 1e-12)
    grad[0] = 1e3
    steps = _steps(0)
    state = ops.adamw8_state(params[0])
    plan = ops.adamw8_plan(params, [state[0]], [state[1]], [state[2]],
                           [state[3]], steps)
    for _ in range(4):
        ops.adamw_step(plan, [grad], lr=1e-3)
        root = ops.adamw8_values(state[2], state[3])
        assert bool((root > 0).all())
        # Each step moves a parameter by lr at most times what the momenta
        # allow, (1 - beta1) / sqrt(1 - beta2) = 3.2: nothing is thrown.
    assert float(params[0].abs().max()) < 4 * 1e-3 * 3.3


def test_nan_and_infinity_stay_where_they_are():
    for make in ("32", "8"):
        params = [torch.ones(64)]
        grad = torch.ones(64)
        grad[3], grad[40] = math.nan, math.inf
        if make == "32":
            plan = ops.adamw_plan(params, [torch.zeros(64)],
                                  [torch.zeros(64)], _steps(0))
        else:
            plan = ops.adamw8_plan(
                params, *[[x] for x in ops.adamw8_state(params[0])], _steps(0))
        for _ in range(2):
            ops.adamw_step(plan, [grad], lr=1e-3)
        bad = torch.zeros(64, dtype=torch.bool)
        bad[[3, 40]] = True
        assert torch.equal(~params[0].isfinite(), bad)


def test_averages_follow_in_8_bits():
    # r of a constant gradient: with unbiased rounding the mean over many
    # elements follows sqrt(1 - beta2^t) |g|, though one step moves r by far
    # less than half a quantum. Its quantum is at most an eighth, so one
    # rounding's spread is at most r / 16; a rounding lasts 1/(1 - beta2^.5)
    # steps or so, so t of them add up to at most sqrt(t) r / 16 = 0.9 r each,
    # and the mean over 32768 elements to 0.005 r: 4 of these, and as much for
    # the bias of a square's root (half the variance).
    n, t = 32768, 200
    params = [torch.zeros(n)]
    state = ops.adamw8_state(params[0])
    plan = ops.adamw8_plan(params, *[[x] for x in state], _steps(0), seed=11)
    grad = torch.full((n,), 0.37)
    for _ in range(t):
        ops.adamw_step(plan, [grad], lr=1e-5)
    root = float(ops.adamw8_values(state[2], state[3]).mean())
    assert root == pytest.approx(0.37 * (1 - 0.999 ** t) ** .5, rel=0.04)
    m = float(ops.adamw8_values(state[0], state[1]).mean())
    assert m == pytest.approx(0.37, rel=0.01)


# ---------------------------------------------------------------------------- #
# Refusals


def _plan_args(n=40, bits=8):
    p = torch.zeros(n)
    if bits == 32:
        return [[p], [torch.zeros(n)], [torch.zeros(n)], _steps(0)]
    return [[p], *[[x] for x in ops.adamw8_state(p)], _steps(0)]


@pytest.mark.parametrize("bits,place,value", [
    (32, 0, [torch.zeros(40, dtype=torch.float64)]),
    (32, 0, [torch.zeros(80)[::2]]),
    (32, 0, []),
    (32, 1, [torch.zeros(41)]),
    (32, 1, [torch.zeros(40, dtype=torch.bfloat16)]),
    (32, 1, []),
    (32, 2, [torch.zeros(80)[::2]]),
    (32, 3, torch.zeros(1)),
    (32, 3, torch.zeros(2, dtype=torch.int32)),
    (8, 1, [torch.zeros(40)]),
    (8, 2, [torch.zeros(2, dtype=torch.uint8)]),
    (8, 2, [torch.zeros(1, dtype=torch.uint8).view(torch.float8_e8m0fnu)]),
    (8, 4, [torch.zeros(3, dtype=torch.uint8).view(torch.float8_e8m0fnu)]),
])
def test_plan_refuses(bits, place, value):
    args = _plan_args(bits=bits)
    make = ops.adamw_plan if bits == 32 else ops.adamw8_plan
    make(*args)
    args[place] = value
    with pytest.raises(RuntimeError):
        make(*args)


def test_plan_refuses_another_number_of_places():
    for places in ([], [0, 1]):
        with pytest.raises(RuntimeError, match="places"):
            ops.adamw8_plan(*_plan_args(), places=places)
    ops.adamw8_plan(*_plan_args(), places=[3])


def test_plan_refuses_shared_memory():
    flat = torch.zeros(100)
    other = lambda: [torch.zeros(40), torch.zeros(40)]  # noqa: E731
    with pytest.raises(RuntimeError, match="share memory"):
        ops.adamw_plan([flat[:40], flat[39:79]], other(), other(),
                       _steps(0, 0))
    with pytest.raises(RuntimeError, match="share memory"):
        ops.adamw_plan([flat[:40]], [flat[20:60]], [torch.zeros(40)],
                       _steps(0))
    ops.adamw_plan([flat[:40], flat[40:80]], other(), other(), _steps(0, 0))


@pytest.mark.parametrize("change", [
    dict(grads=[]), dict(grads=[torch.zeros(41)]),
    dict(grads=[torch.zeros(40, dtype=torch.float64)]),
    dict(grads=[torch.zeros(40).to_sparse()]),
    dict(lr=-1.), dict(lr=math.nan), dict(lr=math.inf), dict(beta1=1.),
    dict(beta2=-0.1), dict(eps=0.), dict(weight_decay=math.nan),
    dict(norm=torch.ones(())), dict(max_norm=1.),
    dict(norm=torch.ones(()), max_norm=0.),
    dict(norm=torch.ones((), dtype=torch.float64), max_norm=1.),
    dict(norm=torch.ones(2), max_norm=1.)])
def test_step_refuses(change):
    args = _plan_args(bits=32)
    plan = ops.adamw_plan(*args)
    with pytest.raises(RuntimeError):
        ops.adamw_step(plan, **{"grads": [torch.ones(40)], "lr": 0.1,
                                **change})
    assert int(args[3]) == 0 and torch.equal(args[0][0], torch.zeros(40))


def test_step_refuses_what_it_writes_as_input():
    args = _plan_args(bits=32)
    plan = ops.adamw_plan(*args)
    for shared in (args[0][0], args[1][0]):
        with pytest.raises(RuntimeError, match="shares memory"):
            ops.adamw_step(plan, [shared], lr=0.1)
    with pytest.raises(RuntimeError, match="shares memory"):
        ops.adamw_step(plan, [torch.ones(40)], lr=0.1,
                       norm=args[2][0][5], max_norm=1.)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_moved(bits):
    args, want = (_plan_args(bits=bits) for _ in range(2))
    make = ops.adamw_plan if bits == 32 else ops.adamw8_plan
    plan, still = make(*args), make(*want)
    for _ in range(3):
        args[0][0].data = args[0][0].data.clone()
        for one in (plan, still):
            ops.adamw_step(one, [torch.arange(40.)], lr=0.1)
    assert torch.equal(args[0][0], want[0][0])
    # What the new memory holds is not its gradient or its norm.
    for change in (lambda new: dict(grads=[new]),
                   lambda new: dict(norm=new[3], max_norm=1.)):
        args[0][0].data = new = torch.ones(40)
        with pytest.raises(RuntimeError, match="shares memory"):
            ops.adamw_step(plan, **{"grads": [torch.ones(40)], "lr": 0.1,
                                    **change(new)})


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_in_another_order_are_refused(bits):
    # Their states stay in the old one: elements would meet others' states.
    p = torch.randn(4, 3, 5, 5)
    state = (ops.adamw8_state(p) if bits == 8 else
             [torch.zeros_like(p) for _ in range(2)])
    make = ops.adamw_plan if bits == 32 else ops.adamw8_plan
    plan = make([p], *[[x] for x in state], _steps(0))
    ops.adamw_step(plan, [torch.ones(4, 3, 5, 5)], lr=0.1)
    p.data = p.data.to(memory_format=torch.channels_last)
    before = p.clone()
    with pytest.raises(RuntimeError, match="strides"):
        ops.adamw_step(plan, [torch.ones(4, 3, 5, 5)], lr=0.1)
    assert torch.equal(p, before)


def test_parameters_that_moved_into_gaps_are_refused():
    args = _plan_args(n=4, bits=32)
    plan = ops.adamw_plan(*args)
    whole = torch.arange(8.)
    args[0][0].data = whole[::2]
    with pytest.raises(RuntimeError, match="fill its memory"):
        ops.adamw_step(plan, [torch.ones(4)], lr=0.1)
    assert torch.equal(whole, torch.arange(8.)) and int(args[3]) == 0
    args[0][0].data = torch.ones(3)
    with pytest.raises(RuntimeError):
        ops.adamw_step(plan, [torch.ones(3)], lr=0.1)


def test_views_that_negate():
    # The imaginary part of a conjugate: its memory holds the opposite numbers.
    def minus(x):
        out = torch.complex(torch.zeros_like(x), -x).conj().imag
        assert out.is_neg() and torch.equal(out, x)
        return out

    def new():
        return [torch.ones(1, device="cpu") for _ in range(3)]
    steps = torch.zeros(1, dtype=torch.int32, device="cpu")
    for k in range(3):
        p, m, v = (minus(x) if i == k else x for i, x in enumerate(new()))
        with pytest.raises(RuntimeError, match="negates"):
            ops.adamw_plan([p], [m], [v], steps)
    p, m, v = new()
    plan = ops.adamw_plan([p], [m], [v], steps)
    five = torch.full((1,), 5., device="cpu")
    with pytest.raises(RuntimeError, match="negates"):
        ops.adamw_step(plan, [five], lr=0.1, norm=minus(five), max_norm=1.)
    # Gradients are only read: they may be.
    assert float(ops.grad_norm([minus(five)])) == 5
    ops.adamw_step(plan, [minus(five)], lr=0.1, beta1=0.5)
    assert float(m) == 3 and int(steps) == 1


def test_16_bit_parameters_refuse_other_gradients():
    p = torch.zeros(8, dtype=torch.bfloat16)
    plan = ops.adamw_plan([p], [torch.zeros(8)], [torch.zeros(8)], _steps(0))
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(RuntimeError):
            ops.adamw_step(plan, [torch.ones(8, dtype=dtype)], lr=0.1)


def test_grad_norm_refuses():
    for bad in ([], [torch.zeros(3, dtype=torch.int32)],
                [torch.zeros(3).to_sparse()]):
        with pytest.raises(RuntimeError):
            ops.grad_norm(bad)


def test_grad_norm_refuses_to_lose_a_gradient():
    x = torch.ones(4, requires_grad=True)
    for tensors in ([x], [torch.ones(3), x * 2]):
        with pytest.raises(RuntimeError, match="no_grad"):
            ops.grad_norm(tensors)
    with torch.no_grad():
        assert float(ops.grad_norm(x)) == 2
    assert float(ops.grad_norm(x.detach())) == 2
    assert not ops.grad_norm(torch.ones(3)).requires_grad


# ---------------------------------------------------------------------------- #
# Optimizer


def _model(channels_last=False, seed=0):
    torch.manual_seed(seed)
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3), torch.nn.Flatten(),
                                torch.nn.Linear(8 * 36, 10))
    return model.to(memory_format=torch.channels_last) if channels_last \
        else model


def _train(model, optimizer, steps, seed=0):
    gen = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        optimizer.zero_grad()
        model(torch.randn(4, 3, 8, 8, generator=gen)).square().mean().backward()
        optimizer.step()


def test_optimizer_matches_torch():
    mine, other = _model(), _model()
    a = AdamW(mine.parameters(), lr=1e-3, weight_decay=0.1)
    b = torch.optim.AdamW(other.parameters(), lr=1e-3, weight_decay=0.1)
    _train(mine, a, 10)
    _train(other, b, 10)
    for p, q in zip(mine.parameters(), other.parameters()):
        # Ten steps of 1e-3, each off by 20 u of itself or so, and by the
        # gradients' own differences.
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-6)


def test_optimizer_clips_as_torch_does():
    mine, other = _model(), _model()
    a = AdamW(mine.parameters(), max_norm=0.01)
    b = torch.optim.AdamW(other.parameters())
    x = torch.randn(4, 3, 8, 8)
    for model in (mine, other):
        model(x).square().mean().backward()
    norm = torch.nn.utils.clip_grad_norm_(other.parameters(), 0.01)
    assert float(norm) > 0.01
    a.step()
    b.step()
    for p, q in zip(mine.parameters(), other.parameters()):
        # clip_grad_norm_ adds 1e-6 to the norm; m / sqrt(v) hardly sees it.
        torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("channels_last", [False, True])
def test_checkpoint_goes_on_alike(bits, channels_last):
    whole = _model(channels_last)
    opt = AdamW(whole.parameters(), state_bits=bits, rounding_seed=3)
    _train(whole, opt, 3)
    file = io.BytesIO()
    torch.save({"m": whole.state_dict(), "o": opt.state_dict()}, file)
    file.seek(0)
    saved = torch.load(file, weights_only=True)
    again = _model(channels_last, seed=9)
    again.load_state_dict(saved["m"])
    opt2 = AdamW(again.parameters(), rounding_seed=3)
    opt2.load_state_dict(saved["o"])
    copied = copy.deepcopy((whole, opt))
    for model, optimizer in ((whole, opt), (again, opt2), copied):
        _train(model, optimizer, 3, seed=1)
    for p, q, w in zip(whole.parameters(), again.parameters(),
                       copied[0].parameters()):
        assert torch.equal(p, q) and torch.equal(p, w)
    assert int(opt2.state[next(again.parameters())]["step"]) == 6


def test_checkpoint_into_another_memory_order():
    first = _model(True)
    opt = AdamW(first.parameters(), state_bits=8)
    _train(first, opt, 3)
    second = _model(False)
    second.load_state_dict(first.state_dict())
    opt2 = AdamW(second.parameters(), state_bits=8)
    opt2.load_state_dict(opt.state_dict())
    for p, q in zip(first.parameters(), second.parameters()):
        for name in ("exp_avg", "exp_avg_root"):
            x, y = (ops.adamw8_values(s[name], s[name + "_scale"])
                    for s in (opt.state[p], opt2.state[q]))
            # To nearest: half of e4m3's step, or of its least step.
            assert bool(((x - y).abs() <= 2. ** -4 * x.abs()
                         + 2. ** -18 * x.abs().max()).all())
    _train(second, opt2, 1)


def test_loads_torchs_state():
    first, second = _model(), _model()
    opt = torch.optim.AdamW(first.parameters())
    _train(first, opt, 3)
    second.load_state_dict(first.state_dict())
    opt2 = AdamW(second.parameters())
    opt2.load_state_dict(opt.state_dict())
    _train(first, opt, 2, seed=1)
    _train(second, opt2, 2, seed=1)
    for p, q in zip(first.parameters(), second.parameters()):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-6)


def test_loads_only_what_it_can_go_on_with():
    model = _model()
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        other = torch.optim.AdamW(model.parameters(), **kw)
        _train(model, other, 1)
        with pytest.raises(ValueError):
            AdamW(model.parameters()).load_state_dict(other.state_dict())
    sgd = torch.optim.SGD(model.parameters(), lr=0.5, momentum=0.9)
    _train(model, sgd, 1)
    with pytest.raises(ValueError):
        AdamW(model.parameters()).load_state_dict(sgd.state_dict())
    # Without states there is nothing to go on with but the settings.
    opt = AdamW(model.parameters(), eps=1e-6, state_bits=8)
    opt.load_state_dict(torch.optim.SGD(model.parameters(),
                                        lr=0.5).state_dict())
    assert opt.param_groups[0]["lr"] == 0.5
    assert opt.param_groups[0]["eps"] == 1e-6
    assert opt.param_groups[0]["state_bits"] == 8
    _train(model, opt, 1)


def test_optimizer_refuses():
    model = _model()
    with pytest.raises(tools.UserException):
        AdamW(model.parameters(), state_bits=16)
    with pytest.raises(tools.UserException):
        AdamW(model.parameters(), max_norm=0.)
    opt = AdamW(model.parameters())
    _train(model, opt, 1)
    state = opt.state_dict()
    state["param_groups"][0]["state_bits"] = 8
    with pytest.raises(ValueError):
        AdamW(model.parameters()).load_state_dict(state)
    with pytest.raises(ValueError):
        AdamW(list(model.parameters())[1:]).load_state_dict(opt.state_dict())


def test_loading_does_not_stretch_states():
    model = _model()
    opt = AdamW(model.parameters())
    _train(model, opt, 1)
    state = opt.state_dict()
    state["state"][0]["exp_avg"] = torch.zeros(1)
    with pytest.raises(ValueError, match="shape"):
        AdamW(model.parameters()).load_state_dict(state)


@pytest.mark.parametrize("bits", [32, 8])
def test_loading_shares_nothing(bits):
    first, second = _model(), _model()
    opt = AdamW(first.parameters(), state_bits=bits)
    _train(first, opt, 2)
    second.load_state_dict(first.state_dict())
    opt2 = AdamW(second.parameters(), state_bits=bits)
    opt2.load_state_dict(opt.state_dict())
    _train(first, opt, 3, seed=1)  # while the other waits
    _train(second, opt2, 3, seed=1)
    assert int(opt2.state[next(second.parameters())]["step"]) == 5
    for p, q in zip(first.parameters(), second.parameters()):
        assert torch.equal(p, q)


def test_loads_no_decay_that_is_not_decoupled():
    model = _model()
    for other in (torch.optim.Adam, torch.optim.SGD):
        opt = other(model.parameters(), lr=0.1, weight_decay=0.1)
        with pytest.raises(ValueError, match="decoupled"):
            AdamW(model.parameters()).load_state_dict(opt.state_dict())
    other = AdamW(model.parameters(), weight_decay=0.3)
    other.load_state_dict(torch.optim.Rprop(model.parameters()).state_dict())
    assert other.param_groups[0]["weight_decay"] == 0.3  # it has none to give
    for opt in (torch.optim.AdamW(model.parameters(), weight_decay=0.1),
                torch.optim.Adam(model.parameters())):
        _train(model, opt, 1)
        mine = AdamW(model.parameters())
        mine.load_state_dict(opt.state_dict())
        decay = opt.param_groups[0]["weight_decay"]
        assert mine.param_groups[0]["weight_decay"] == decay
        # From then on it is this optimizer's, with the decay that it has.
        mine.param_groups[0]["weight_decay"] = 0.2
        again = AdamW(model.parameters())
        again.load_state_dict(mine.state_dict())
        assert again.param_groups[0]["weight_decay"] == 0.2


@pytest.mark.parametrize("bits", [32, 8])
def test_load_hooks_see_the_states(bits):
    model = _model()
    opt = AdamW(model.parameters(), state_bits=bits)
    _train(model, opt, 3)
    saved, seen = opt.state_dict(), []

    def before(_, given):
        seen.append(sorted(given["state"]))
        states = {i: {**s, "step": torch.tensor(7)}
                  for i, s in given["state"].items()}
        return {**given, "state": states}

    def after(optimizer):
        seen.append([int(optimizer.state[p]["step"])
                     for p in model.parameters()])

    opt2 = AdamW(model.parameters())
    opt2.register_load_state_dict_pre_hook(before)
    opt2.register_load_state_dict_post_hook(after)
    for _ in range(2):
        opt2.load_state_dict(saved)
    assert seen == [[0, 1, 2, 3], [7] * 4] * 2
    _train(model, opt2, 1)
    assert int(opt2.state[next(model.parameters())]["step"]) == 8
    # What is refused leaves the optimizer as it was.
    saved["param_groups"][0]["state_bits"] = 40 - bits
    with pytest.raises(ValueError):
        opt2.load_state_dict(saved)
    assert opt2.param_groups[0]["state_bits"] == bits
    assert int(opt2.state[next(model.parameters())]["step"]) == 8


def test_loading_takes_scales_of_the_right_number():
    model = _model()
    opt = AdamW(model.parameters(), state_bits=8)
    _train(model, opt, 1)
    for name in ("exp_avg_scale", "exp_avg_root_scale"):
        saved = copy.deepcopy(opt.state_dict())
        saved["state"][2][name] = saved["state"][2][name][1:]
        with pytest.raises(ValueError, match=name):
            AdamW(model.parameters()).load_state_dict(saved)


@pytest.mark.parametrize("setting", [
    dict(lr=-1.), dict(lr=math.nan), dict(betas=(1., 0.9)),
    dict(betas=(0.9, -0.1)), dict(eps=0.), dict(weight_decay=-1.),
    dict(max_norm=-1.), dict(max_norm=math.inf), dict(max_norm=1e-40),
    dict(max_norm=math.nan)])
def test_settings_that_no_step_takes_are_refused_at_once(setting):
    model = _model()
    with pytest.raises(tools.UserException):
        AdamW(model.parameters(), **setting)
    if "max_norm" in setting:
        return
    first, *others = model.parameters()
    opt = AdamW([first])
    with pytest.raises(tools.UserException):
        opt.add_param_group({"params": others, **setting})
    assert len(opt.param_groups) == 1
    saved = AdamW(model.parameters()).state_dict()
    saved["param_groups"][0].update(setting)
    with pytest.raises(ValueError, match="out of range"):
        AdamW(model.parameters()).load_state_dict(saved)


def test_values_refuse():
    codes, scales, *_ = ops.adamw8_state(torch.zeros(100))
    assert torch.equal(ops.adamw8_values(codes, scales), torch.zeros(100))
    for a, b in ((codes.float(), scales), (codes[::2], scales[:2]),
                 (codes, scales[:3]), (codes, scales.float())):
        with pytest.raises(RuntimeError):
            ops.adamw8_values(a, b)


def test_any_iterable_of_tensors():
    args = _plan_args(bits=32)
    plan = ops.adamw_plan(*args)
    ops.adamw_step(plan, (g for g in [torch.ones(40)]), lr=0.1)
    ops.adamw_step(plan, (torch.ones(40),), lr=0.1)
    assert int(args[3]) == 2
    assert float(ops.grad_norm(t for t in [torch.ones(9)])) == 3


def test_schedulers_reach_the_step():
    p = torch.nn.Parameter(torch.ones(()))
    opt = AdamW([p], lr=1., weight_decay=0.)
    schedule = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.)
    p.grad = torch.ones(())
    opt.step()
    schedule.step()
    before = p.detach().clone()
    assert float(before) == pytest.approx(0., abs=1e-6)
    opt.step()
    assert torch.equal(p, before)


def test_groups_with_their_own_settings():
    model = _model()
    params = list(model.parameters())
    opt = AdamW([{"params": params[:2], "state_bits": 8, "lr": 0.},
                 {"params": params[2:]}], lr=1e-2)
    before = [p.detach().clone() for p in params]
    _train(model, opt, 1)
    assert all(torch.equal(a, b) for a, b in zip(before[:2], params[:2]))
    assert not any(torch.equal(a, b) for a, b in zip(before[2:], params[2:]))
    assert "exp_avg_root" in opt.state[params[0]]
    opt.state.clear()
    _train(model, opt, 1)
    assert int(opt.state[params[0]]["step"]) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_states_that_are_cleared_or_replaced(bits):
    whole, other = _model(), _model()
    opt = AdamW(whole.parameters(), state_bits=bits)
    opt2 = AdamW(other.parameters(), state_bits=bits)
    for model, optimizer in ((whole, opt), (other, opt2)):
        _train(model, optimizer, 2)
    params, params2 = list(whole.parameters()), list(other.parameters())
    # Through the state and through load_state_dict.
    names = [k for k in opt.state[params[2]] if k != "step"]
    replaced = {k: v.clone() for k, v in zip(
        names, ops.adamw8_state(params[2]) if bits == 8 else
        [torch.ones_like(params[2]) for _ in range(2)])}
    del opt.state[params[1]]
    opt.state[params[2]].update(replaced)
    opt.state[params[3]]["step"] = 7
    saved = opt2.state_dict()
    del saved["state"][1]
    saved["state"][2].update(replaced)
    saved["state"][3]["step"] = 7
    opt2.load_state_dict(saved)
    for model, optimizer in ((whole, opt), (other, opt2)):
        _train(model, optimizer, 2, seed=1)
    for p, q in zip(params, params2):
        assert torch.equal(p, q)
        x, y = opt.state[p], opt2.state[q]
        assert set(x) == set(y) == {"step", *names}
        assert all(torch.equal(x[k].float(), y[k].float()) for k in x)
    assert [int(opt.state[p]["step"]) for p in params] == [4, 2, 4, 9]
    assert sorted(opt.state_dict()["state"]) == [0, 1, 2, 3]


def test_states_that_are_incomplete_are_refused():
    model = _model()
    opt = AdamW(model.parameters())
    _train(model, opt, 1)
    before = [p.detach().clone() for p in model.parameters()]
    del opt.state[next(model.parameters())]["exp_avg"]
    for _ in range(2):
        with pytest.raises(RuntimeError, match="lacks exp_avg"):
            opt.step()
    assert all(torch.equal(a, b) for a, b in zip(before, model.parameters()))


@pytest.mark.parametrize("bits", [32, 8])
def test_only_parameters_with_a_gradient_have_a_state(bits):
    frozen = torch.nn.Parameter(torch.zeros(9, dtype=torch.float64),
                                requires_grad=False)
    late = torch.nn.Parameter(torch.ones(70))
    model = _model()
    opt = AdamW([frozen, late, *model.parameters()], state_bits=bits)
    _train(model, opt, 2)
    assert not opt.state.get(frozen) and not opt.state.get(late)
    assert sorted(opt.state_dict()["state"]) == [2, 3, 4, 5]
    first = opt.state[next(model.parameters())]["step"]
    late.grad = torch.arange(70.)
    opt.step()
    assert int(opt.state[late]["step"]) == 1
    # What was there has not moved.
    assert opt.state[next(model.parameters())]["step"] is first
    assert int(first) == 3 and not opt.state.get(frozen)
    again = AdamW([frozen, late, *model.parameters()])
    again.load_state_dict(opt.state_dict())
    again.step()
    assert int(again.state[late]["step"]) == 2
    assert not again.state.get(frozen)


@pytest.mark.parametrize("max_norm", [None, 0.1])
def test_rounding_does_not_depend_on_who_else_has_a_gradient(max_norm):
    # Three parameters, the first of them without a gradient at first: one
    # plan, or two.
    def start(late):
        gen = torch.Generator().manual_seed(1)
        params = [torch.nn.Parameter(torch.randn(77, generator=gen))
                  for _ in range(3)]
        opt = AdamW(params, state_bits=8, rounding_seed=5, max_norm=max_norm)
        for k in range(3):
            for i, p in enumerate(params):
                p.grad = None if i == 0 and k < late else torch.randn(
                    77, generator=torch.Generator().manual_seed(10 * i + k))
            opt.step()
        return params, opt

    one, opt = start(0)
    two, opt2 = start(2)
    assert len(opt._plans) == 1 and len(opt2._plans) == 2
    if max_norm is None:  # (the norm is over all that are there)
        for p, q in zip(one[1:], two[1:]):
            assert torch.equal(p, q)
            x, y = opt.state[p], opt2.state[q]
            assert all(torch.equal(x[k].float(), y[k].float()) for k in x)
    # In one plan again, and with the same norm bit by bit.
    merged = copy.deepcopy((two, opt2))
    for params, optimizer in ((two, opt2), merged):
        for i, p in enumerate(params):
            p.grad = torch.full((77,), 0.1 * i + 0.01)
        optimizer.step()
    assert len(opt2._plans) == 2 and len(merged[1]._plans) == 1
    for p, q in zip(two, merged[0]):
        assert torch.equal(p, q)
        x, y = opt2.state[p], merged[1].state[q]
        assert all(torch.equal(x[k].float(), y[k].float()) for k in x)


def test_registry():
    p = [torch.nn.Parameter(torch.zeros(4))]
    opt = build_optimizer("adamw", ["state-bits:8", "clip-norm:2",
                                    "weight-decay:0.5", "rounding-seed:4"],
                          p, 0.25)
    assert isinstance(opt, AdamW) and opt.max_norm == 2
    assert opt.rounding_seed == 4
    group = opt.param_groups[0]
    assert group["state_bits"] == 8 and group["weight_decay"] == 0.5
    assert group["lr"] == 0.25
    assert build_optimizer("adamw", [], p, 1.).max_norm is None


@pytest.mark.parametrize("args", [[], ["state-bits:8", "clip-norm:0.5"]])
def test_engine_steps_and_resumes(args):
    def engine():
        exp = experiments.instantiate("mnist", ["batch-size:16"])
        return Engine(exp, "krum", WorkerGroup(5, device="cpu"), nbbyzwrks=1,
                      optimizer="adamw", optimizer_args=args, seed=5)
    one, two = engine(), engine()
    for _ in range(3):
        assert math.isfinite(one.step())
    file = io.BytesIO()
    torch.save(one.state_dict(), file)
    file.seek(0)
    two.load_state_dict(torch.load(file, weights_only=True))
    one.step()
    two.step()
    for p, q in zip(one.params, two.params):
        assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [32, 8])
def test_ranks_stay_alike(tmp_path, bits):
    worker = pathlib.Path(__file__).parent / "adamw_dist_worker.py"
    outs = [tmp_path / f"rank{rank}.pt" for rank in range(2)]
    procs = [subprocess.Popen(
        [sys.executable, str(worker), str(out), f"state-bits:{bits}"],
        env={**os.environ, "RANK": str(rank), "WORLD_SIZE": "2",
             "LOCAL_RANK": str(rank), "MASTER_ADDR": "127.0.0.1",
             "MASTER_PORT": str(29700 + bits), "GLOO_SOCKET_IFNAME": "lo"},
        stdout=subprocess.PIPE, stderr=subprocess.PIPE)
        for rank, out in enumerate(outs)]
    for p in procs:
        _, err = p.communicate(timeout=300)
        assert p.returncode == 0, err.decode()[-2000:]
    one, two = (torch.load(out, weights_only=True) for out in outs)
    for a, b in zip(one, two):
        assert len(a) == len(b) == (4 if bits == 32 else 6)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------------------- #
# The kernels' code


def _waits(lines):
    """For each barrier of a kernel's assembly: whether all loads of the step
    count (the agent-scope ones) that reach it are waited for, or None where
    none reaches it. Loads come back in order, so with `s_waitcnt vmcnt(n)` a
    load is there once n or more others have been issued behind it."""
    blocks, name = {"": []}, ""
    follows = {}
    for line in lines:
        line = line.split(";")[0].strip()
        if re.match(r"\.LBB\w+:", line):
            previous, name = name, line[:-1]
            blocks[name] = []
            follows.setdefault(previous, set()).add(name)
        elif line and not line.startswith("."):
            blocks[name].append(line)
            if line.startswith(("s_cbranch", "s_branch")):
                follows.setdefault(name, set()).add(line.split()[1])
                # What stands behind a branch is a block of its own.
                previous, name = name, f"{name}+{len(blocks)}"
                blocks[name] = []
                if line.startswith("s_cbranch"):
                    follows[previous].add(name)
            elif line.startswith("s_endpgm"):
                name = f"{name}+{len(blocks)}"
                blocks[name] = []
    # State: how many others have been issued since (the fewest on any way
    # here), -1 for one that is there, None before it.
    states, barriers, todo = {"": {None}}, {}, [""]
    while todo:
        at = todo.pop()
        out = set()
        for state in states[at]:
            for k, line in enumerate(blocks[at]):
                wait = re.search(r"vmcnt\((\d+)\)", line)
                if re.match(r"global_load_dword v\d+, .* sc1", line):
                    state = 0
                elif re.match(r"(global|buffer|flat)_", line):
                    state = min(state + 1, 64) if state not in (None, -1) \
                        else state
                elif line.startswith("s_waitcnt") and wait and \
                        state not in (None, -1) and int(wait[1]) <= state:
                    state = -1
                elif line.startswith("s_barrier"):
                    barriers.setdefault((at, k), set()).add(state)
            out.add(state)
        for to in follows.get(at, ()):
            if not out <= states.setdefault(to, set()):
                states[to] |= out
                todo.append(to)
    return [None if s == {None} else s == {-1} for s in barriers.values()]


def test_waits_are_seen():
    # The reading of the assembly, on the two ways that a load may be left.
    def kernel(*wait):
        return ["s_cbranch_scc0 .LBB0_2", ".LBB0_1:",
                "global_load_dword v1, v2, s[4:5] sc1",
                "global_load_dwordx4 v[4:7], v[8:9], off nt",
                "s_branch .LBB0_3", ".LBB0_2:",
                "global_load_dword v1, v2, s[4:5] sc1",
                "global_load_dwordx4 v[4:7], v[8:9], off nt",
                "global_load_dwordx4 v[4:7], v[8:9], off nt",
                ".LBB0_3:", *wait, "s_barrier", "s_waitcnt vmcnt(0)",
                "s_endpgm"]
    assert _waits(kernel("s_waitcnt vmcnt(1)")) == [True]
    assert _waits(kernel("s_waitcnt vmcnt(2)")) == [False]
    assert _waits(kernel()) == [False]
    assert _waits(["s_barrier", "s_endpgm"]) == [None]


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="needs hipcc")
def test_step_counts_are_read_before_the_barrier(tmp_path):
    # Behind the barrier a workgroup says that it has read the count, and the
    # last to say so writes it: a wave's load that the barrier does not find
    # waited for might get the next step's.
    out = tmp_path / "adamw.s"
    subprocess.run(["hipcc", "-S", "--cuda-device-only",
                    *ops_build._compile_flags(),
                    str(ops_build.CSRC / "adamw_kernels.hip"), "-o", str(out)],
                   check=True, stderr=subprocess.DEVNULL)
    kernels = re.findall(r"^(\S*update_kernel\S*):(.*?)^\.Lfunc_end",
                         out.read_text(), re.M | re.S)
    assert len(kernels) == 3
    for name, text in kernels:
        found = _waits(text.splitlines())
        assert found and all(found), f"{name}: {found}"
