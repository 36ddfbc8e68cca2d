"""Optimizer kernels on the GPU: against 64 bits, against the plain forms bit
by bit where these are exact, and in the ways that they are called (streams,
graphs, layouts, long lists, large tensors)."""

import io
import math

import pytest
import torch

import adamw_oracle as oracle
from aggregathor_amd import experiments, ops
from aggregathor_amd.graph import Engine, bind_grad_views
from aggregathor_amd.ops import adamw_reference as R
from aggregathor_amd.optim import AdamW
from aggregathor_amd.parallel import WorkerGroup

pytestmark = pytest.mark.gpu

# Around a quad, a group, a workgroup's part, and several of these.
SIZES = [1, 3, 4, 5, 31, 32, 33, 127, 1025, 4095, 4096, 4097, 0, 12289, 70001]
# Past the size from which 8-bit states take larger parts, in all.
LARGE = [2047, 2048, 1, 2049, 33, 2200001]
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.1)
TYPES = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
         (torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16)]


@pytest.fixture(autouse=True)
def _native():
    assert ops.hip_available(), "HIP extension must be importable on a GPU box"


def _tensors(sizes, dtype=torch.float32, seed=0, scale=1.):
    gen = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(n, generator=gen)).to(dtype) for n in sizes]


def _state32(sizes, seed=1):
    return ([0.1 * t for t in _tensors(sizes, seed=seed)],
            [0.02 * t.square() for t in _tensors(sizes, seed=seed + 1)])


def _state8(sizes, seed=1):
    m, v = _state32(sizes, seed)
    out = [R.nearest8(x, False) + R.nearest8(y.sqrt(), True)
           for x, y in zip(m, v)]
    return [list(column) for column in zip(*out)]


def _cuda(x):
    return [t.cuda() for t in x]


def _packed(tensors, lead=0):
    """The tensors back to back, as views into one buffer on the GPU that
    begins `lead` elements before them."""
    flat = torch.cat([torch.zeros(lead, dtype=tensors[0].dtype)] +
                     list(tensors)).cuda()
    out, at = [], lead
    for t in tensors:
        out.append(flat[at:at + t.numel()])
        at += t.numel()
    return out, flat


def _equal(a, b):
    """Bit by bit, NaN equal to NaN."""
    a, b = a.detach().cpu().float(), b.detach().cpu().float()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(
        a.nan_to_num(7.), b.nan_to_num(7.))


def _check_states(a, b, what=""):
    """8-bit states of the kernel against the plain form's, bit by bit."""
    assert all(_equal(x, y) for x, y in zip(a, b)), what


# ---------------------------------------------------------------------------- #
# Norm


@pytest.mark.parametrize("lead", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
def test_grad_norm(dtype, lead):
    host = _tensors(SIZES, dtype)
    want = sum(float(g.double().square().sum()) for g in host) ** .5
    together, _ = _packed(host, lead)
    for grads in (_cuda(host), together, together[::-1]):
        got = ops.grad_norm(grads)
        assert got.dtype == torch.float32 and got.shape == ()
        # Sums in 64 bits: only the rounding to fp32 is left.
        assert abs(float(got) - want) <= 2 * oracle.U * want
        assert torch.equal(got, ops.grad_norm(grads))


def test_grad_norm_of_many_and_mixed():
    host = [t.to(d) for t, d in zip(
        _tensors([n % 97 for n in range(1000)]),
        [torch.float32, torch.bfloat16, torch.float16, torch.float32] * 250)]
    host[7] = host[7].repeat(10, 1).t()
    want = sum(float(g.double().square().sum()) for g in host) ** .5
    grads = _cuda(host)
    grads[9] = torch.zeros(3, 50, device="cuda")[:, ::2]  # gaps
    grads[11] = torch.ones(1, device="cuda").expand(9)    # one for all
    want = sum(float(g.double().square().sum()) for g in grads) ** .5
    assert abs(float(ops.grad_norm(grads)) - want) <= 2 * oracle.U * want


@pytest.mark.parametrize("count", [176, 199, 200, 201, 400, 401])
def test_grad_norm_of_separate_tensors(count):
    # Around one launch's spans, and two's.
    host = _tensors([1 + 37 * i % 211 for i in range(count)])
    grads = _packed([t for g in host for t in (g, torch.full((1,), 99.))])[0]
    want = sum(float(g.double().square().sum()) for g in host) ** .5
    for _ in range(2):
        got = float(ops.grad_norm(grads[::2]))  # a gap behind each
        assert abs(got - want) <= 2 * oracle.U * want


def test_grad_norm_extremes():
    for value, n, want in ((0., 5, 0.), (1e30, 4, 2e30), (1e-30, 4, 2e-30),
                           (3e38, 1, 3e38), (math.nan, 3, math.nan),
                           (-math.inf, 3, math.inf)):
        got = float(ops.grad_norm(torch.full((n,), value, device="cuda")))
        assert got == pytest.approx(want, rel=1e-6, nan_ok=True)
    assert float(ops.grad_norm([torch.zeros(0, device="cuda")])) == 0
    three = torch.full((9,), 1., device="cuda")
    assert float(ops.grad_norm([three] * 4)) == 6


def test_grad_norm_refuses_to_lose_a_gradient():
    x = torch.ones(4, device="cuda", requires_grad=True)
    for tensors in ([x], [torch.ones(3, device="cuda"), x * 2]):
        with pytest.raises(RuntimeError, match="no_grad"):
            ops.grad_norm(tensors)
    with torch.no_grad():
        assert float(ops.grad_norm(x)) == 2
    assert float(ops.grad_norm(x.detach())) == 2
    assert not ops.grad_norm(torch.ones(3, device="cuda")).requires_grad


def test_grad_norm_large():
    # Past 2^32 bytes, and past 2^31 elements in bf16.
    n = (1 << 31) + 4097
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[-1], x[0], x[1 << 31] = 3., 4., 12.
    assert float(ops.grad_norm(x)) == 13.


# ---------------------------------------------------------------------------- #
# Step


@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
@pytest.mark.parametrize("p_dtype,g_dtype", TYPES)
def test_step32(p_dtype, g_dtype, max_norm):
    params, grads = _tensors(SIZES, p_dtype), _tensors(SIZES, g_dtype, 5, 0.3)
    m, v = _state32(SIZES)
    counts = [(37 * i) % 1000 for i in range(len(SIZES))]
    s = 1. if max_norm is None else oracle.clip_factor(grads, max_norm)[1]
    want = [oracle.step(*x, t + 1, **HYPER, s=s)
            for *x, t in zip(params, grads, m, v, counts)]
    # Parameters and states of their own, gradients packed at an odd start.
    p, m, v = _cuda(params), _cuda(m), _cuda(v)
    g, _ = _packed(grads, 1)
    steps = torch.tensor(counts, dtype=torch.int32, device="cuda")
    ops.adamw_step(ops.adamw_plan(p, m, v, steps), g, **HYPER,
                   norm=None if max_norm is None else ops.grad_norm(g),
                   max_norm=max_norm)
    assert steps.tolist() == [t + 1 for t in counts]
    for i, (values, bounds) in enumerate(want):
        bounds = (oracle.rounded(bounds[0], values[0], p_dtype), *bounds[1:])
        for name, got, x, b in zip("pmv", (p[i], m[i], v[i]), values, bounds):
            oracle.check(got, x, b, f"{name} of {SIZES[i]}")


@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("p_dtype,g_dtype", TYPES)
@pytest.mark.parametrize("sizes", [SIZES, LARGE])
def test_step8(sizes, p_dtype, g_dtype, max_norm):
    params, grads = _tensors(sizes, p_dtype), _tensors(sizes, g_dtype, 5, 0.3)
    state = _state8(sizes)
    counts = [(37 * i) % 1000 for i in range(len(sizes))]
    values = [(R.values8(a, b), R.values8(c, d).square())
              for a, b, c, d in zip(*state)]
    s = 1. if max_norm is None else oracle.clip_factor(grads, max_norm)[1]
    want = [oracle.step(a, b, *mv, t + 1, **HYPER, s=s)
            for a, b, mv, t in zip(params, grads, values, counts)]
    p, g = _cuda(params), _packed(grads, 1)[0]
    own = [_cuda(column) for column in state]
    steps = torch.tensor(counts, dtype=torch.int32, device="cuda")
    ops.adamw_step(ops.adamw8_plan(p, *own, steps, seed=77), g, **HYPER,
                   norm=None if max_norm is None else ops.grad_norm(g),
                   max_norm=max_norm)
    # The plain form on the CPU: states bit by bit.
    ops.adamw_step(ops.adamw8_plan(
        params, *state, torch.tensor(counts, dtype=torch.int32), seed=77),
        grads, **HYPER, max_norm=max_norm,
        norm=None if max_norm is None else ops.grad_norm(grads))
    assert steps.tolist() == [t + 1 for t in counts]
    for i, (x, bounds) in enumerate(want):
        what = f"of {sizes[i]}"
        oracle.check(p[i], x[0], oracle.rounded(bounds[0], x[0], p_dtype),
                     "p " + what)
        _check_states([c[i] for c in own], [c[i] for c in state], what)
        m, ms, r, rs = (column[i] for column in own)
        oracle.check8(m, ms, ops.adamw8_values(m, ms), x[1], False, "m " + what)
        oracle.check8(r, rs, ops.adamw8_values(r, rs), x[2].sqrt(), True,
                      "r " + what)


def test_step8_states_at_odd_starts_leave_their_neighbours():
    sizes = [33, 70, 4099]
    state = _state8(sizes)
    flats = [_packed([t.view(torch.uint8) for t in column], 3)
             for column in state]
    kinds = (torch.float8_e4m3fn, torch.float8_e8m0fnu) * 2
    views = [[t.view(kind) for t in column]
             for (column, _), kind in zip(flats, kinds)]
    params, grads = _tensors(sizes), _tensors(sizes, seed=5)
    p, pflat = _packed(params, 1)
    steps = torch.zeros(3, dtype=torch.int32, device="cuda")
    ops.adamw_step(ops.adamw8_plan(p, *views, steps), _cuda(grads), **HYPER)
    ops.adamw_step(ops.adamw8_plan(params, *state,
                                   torch.zeros(3, dtype=torch.int32)),
                   grads, **HYPER)
    whole = []
    for (_, flat), column, kind in zip(flats, state, kinds):
        want = torch.cat([torch.zeros(3, dtype=torch.uint8)] +
                         [t.view(torch.uint8) for t in column])
        whole.append((flat.view(kind), want.view(kind)))
    _check_states([x for x, _ in whole], [x for _, x in whole])
    assert float(pflat[0]) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_nan_infinity_zero_and_denormals(bits):
    n = 192
    grad = torch.ones(n)
    grad[3], grad[40], grad[41] = math.nan, math.inf, -math.inf
    grad[64:96] = 0.
    grad[96:128] = 1e-42
    grad[128:160] = 1e25  # its square overflows
    grad[160:] = 1e-20    # its square is a denormal number
    out = []
    for device in ("cpu", "cuda"):
        p = torch.ones(n, device=device)
        if bits == 8:
            state = [x for x in ops.adamw8_state(p)]
        else:
            state = [torch.zeros(n, device=device) for _ in range(2)]
        make = ops.adamw8_plan if bits == 8 else ops.adamw_plan
        plan = make([p], *[[x] for x in state],
                    torch.zeros(1, dtype=torch.int32, device=device))
        for _ in range(3):
            ops.adamw_step(plan, [grad.to(device)], lr=1e-3)
        out.append([p, *state])
    if bits == 8:
        _check_states(out[1][1:], out[0][1:])
    else:
        assert all(_equal(a, b) for a, b in zip(out[0][1:], out[1][1:]))
    a, b = (x[0].cpu() for x in out)
    assert torch.equal(a.isnan(), b.isnan())
    # Three steps of 1e-3, each off by 40 u of itself at most.
    torch.testing.assert_close(a, b, rtol=1e-6, atol=1e-8, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_are_not_finite(bits, dtype):
    p = torch.tensor([math.nan, math.inf, -math.inf, 1., -0.], device="cuda",
                     dtype=dtype)
    opt = AdamW([p], lr=0.5, weight_decay=0.5, state_bits=bits)
    p.grad = torch.zeros(5, device="cuda", dtype=dtype)
    opt.step()
    assert p[0].isnan()
    assert p[1:].tolist() == [math.inf, -math.inf, 0.75, 0.]


@pytest.mark.parametrize("bits", [32, 8])
def test_plain_form_on_the_gpu(bits, monkeypatch):
    kernel = _small_plan(bits)
    monkeypatch.setenv("AGGREGATHOR_FORCE_EAGER", "1")
    plain = _small_plan(bits)
    assert isinstance(plain[0], R.Plan)
    for plan, params, state, steps, grads in (kernel, plain):
        norm = ops.grad_norm(grads)
        for _ in range(2):
            ops.adamw_step(plan, grads, **HYPER, norm=norm, max_norm=0.5)
    assert torch.equal(kernel[3], plain[3])
    for a, b in zip(kernel[2], plain[2]):
        assert all(_equal(x, y) for x, y in zip(a, b))
    for a, b in zip(kernel[1], plain[1]):
        torch.testing.assert_close(a, b, rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("norm", [0., math.inf, math.nan])
def test_norms_that_are_none(norm):
    p = torch.ones(5, device="cuda")
    m, v = torch.ones(5, device="cuda"), torch.ones(5, device="cuda")
    plan = ops.adamw_plan([p], [m], [v],
                          torch.zeros(1, dtype=torch.int32, device="cuda"))
    ops.adamw_step(plan, [torch.ones(5, device="cuda")], lr=0.1,
                   norm=torch.tensor(norm, device="cuda"), max_norm=1.)
    if math.isnan(norm):
        assert bool(p.isnan().all())
    else:
        want = 0.9 + (0.1 if norm == 0. else 0.)
        torch.testing.assert_close(m, torch.full_like(m, want))


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_and_many_tensors(bits):
    # More tensors than one launch takes, some empty, some without a gradient.
    sizes = [(i * 7) % 50 for i in range(1000)]
    params, grads = _tensors(sizes), _tensors(sizes, seed=5)
    state = _state8(sizes) if bits == 8 else _state32(sizes)
    make = ops.adamw8_plan if bits == 8 else ops.adamw_plan
    p, own = _cuda(params), [_cuda(column) for column in state]
    steps = torch.zeros(1000, dtype=torch.int32, device="cuda")
    present = [i % 3 != 1 and not 448 <= i < 896 for i in range(1000)]
    ops.adamw_step(make(p, *own, steps),
                   [g.cuda() if ok else None for g, ok in zip(grads, present)],
                   **HYPER)
    ops.adamw_step(make(params, *state, torch.zeros(1000, dtype=torch.int32)),
                   [g if ok else None for g, ok in zip(grads, present)],
                   **HYPER)
    assert steps.tolist() == [int(ok) for ok in present]
    for i in range(1000):
        a, b = ([c[i] for c in x] for x in (own, state))
        if bits == 8:
            _check_states(a, b)
        else:
            assert all(_equal(x, y) for x, y in zip(a, b))
    for x, y in zip(p, params):
        torch.testing.assert_close(x.cpu(), y, rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(bits):
    gen = torch.Generator().manual_seed(0)
    shape = (6, 5, 3, 3)
    base = torch.randn(shape, generator=gen)
    grad = torch.randn(shape, generator=gen)
    orders = {"plain": base.clone(),
              "last": base.to(memory_format=torch.channels_last),
              "turned": base.permute(3, 1, 0, 2).contiguous().permute(
                  2, 1, 3, 0)}
    for name, order in orders.items():
        for g in (grad, grad.to(memory_format=torch.channels_last),
                  torch.empty_like(order).copy_(grad)):
            out = []
            for device in ("cpu", "cuda"):
                p = order.to(device, copy=True)  # the step is in place
                assert p.stride() == order.stride()
                opt = AdamW([p], lr=0.1, state_bits=bits)
                for _ in range(2):
                    p.grad = g.to(device)
                    opt.step()
                out.append((p, opt.state[p]))
            (a, x), (b, y) = out
            torch.testing.assert_close(a, b.cpu(), rtol=1e-6, atol=1e-6)
            assert _equal(x["step"], y["step"])
            if bits == 8:
                _check_states(*([s[k] for k in (
                    "exp_avg", "exp_avg_scale", "exp_avg_root",
                    "exp_avg_root_scale")] for s in (y, x)), name)
            else:
                assert all(_equal(x[k], y[k]) for k in x), name


def test_expanded_and_strided_gradients():
    p = [torch.ones(4, 6, device="cuda") for _ in range(2)]
    zeros = lambda: [torch.zeros(4, 6, device="cuda")  # noqa: E731
                     for _ in range(2)]
    m = zeros()
    plan = ops.adamw_plan(p, m, zeros(),
                          torch.zeros(2, dtype=torch.int32, device="cuda"))
    g = [torch.full((1, 1), 2., device="cuda").expand(4, 6),
         torch.arange(48., device="cuda").view(4, 12)[:, ::2]]
    ops.adamw_step(plan, g, lr=0.1, beta1=0.5)
    for a, b in zip(m, g):
        assert torch.equal(a, 0.5 * b)


def test_large_tensor_8():
    # Offsets past 2^32 elements: the last parts against the plain form.
    n = (1 << 32) + 4096 + 33
    tail = 4096 + 33 + 32  # from the group before 2^32
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    state = ops.adamw8_state(p)
    p[-tail:], g[-tail:] = 1., torch.randn(tail).to(torch.bfloat16)
    steps = torch.zeros(1, dtype=torch.int32, device="cuda")
    plan = ops.adamw8_plan([p], *[[x] for x in state], steps, seed=5)
    ops.adamw_step(plan, [g], **HYPER)
    x = g[-tail:].cpu().float()
    m, v = x * (1 - 0.9), x * x * (1 - 0.99)
    bits = R.random_bits(5, 0, 1, tail, "cpu", begin=n - tail)
    groups = -(-tail // 32)
    for codes, scales, values, of, root, chance in (
            (state[0], state[1], m, m, False, bits & 0xFFFF),
            (state[2], state[3], v.sqrt(), v, True, bits >> 16)):
        exponents = R.exponents_of(R._largest(of), root)
        assert torch.equal(scales[-groups:].cpu().view(torch.uint8),
                           exponents.to(torch.uint8))
        want = R.round_by_chance(values, exponents, chance, float(root))
        got = codes[-tail:]
        _check_states((want, scales, got, scales) if root else
                      (got, scales, want, scales),
                      (want, scales, want, scales))
    want, bounds = oracle.step(torch.ones(tail), x, torch.zeros(tail),
                               torch.zeros(tail), 1, **HYPER)
    oracle.check(p[-tail:], want[0], oracle.rounded(
        bounds[0], want[0], torch.bfloat16), "p")
    assert float(p[0]) == 0 and not bool(state[0][:1 << 20].float().any())


def test_large_tensor_32():
    # Past 2^32 bytes of a state, 2^31 elements.
    n = (1 << 31) + 4097
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m, v = (torch.zeros(n, device="cuda") for _ in range(2))
    g[-4097:] = 1.
    plan = ops.adamw_plan([p], [m], [v],
                          torch.zeros(1, dtype=torch.int32, device="cuda"))
    ops.adamw_step(plan, [g], lr=0.5)
    assert torch.equal(m[-4098:].cpu(), torch.cat(
        [torch.zeros(1), torch.full((4097,), 1.) * (1 - 0.9)]))
    assert bool((p[-4097:] == -0.5).all()) and float(p[-4098]) == 0


# ---------------------------------------------------------------------------- #
# How it is called


def _small_plan(bits, device="cuda", seed=0):
    sizes = [100, 5000, 33]
    params = [t.to(device) for t in _tensors(sizes, seed=seed)]
    state = _state8(sizes) if bits == 8 else _state32(sizes)
    state = [[t.to(device) for t in column] for column in state]
    steps = torch.zeros(3, dtype=torch.int32, device=device)
    make = ops.adamw8_plan if bits == 8 else ops.adamw_plan
    grads = [t.to(device) for t in _tensors(sizes, seed=5)]
    return make(params, *state, steps), params, state, steps, grads


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_are_steps(bits):
    plan, params, state, steps, grads = _small_plan(bits)
    eager = _small_plan(bits)

    def one(plan, grads):
        ops.adamw_step(plan, grads, **HYPER, norm=ops.grad_norm(grads),
                       max_norm=0.5)

    # Two graphs on the same plan, replayed in turn.
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one(plan, grads)
        graphs.append(graph)
    assert steps.tolist() == [0, 0, 0]
    for k in range(6):
        graphs[k % 2].replay()
        one(eager[0], eager[4])
        torch.cuda.synchronize()
        assert torch.randn(1000, device="cuda").sum().isfinite()
        for g in grads + eager[4]:
            g.mul_(-0.9)
        assert torch.equal(steps, eager[3])
        for a, b in zip(params, eager[1]):
            assert torch.equal(a, b)
        for a, b in zip(state, eager[2]):
            assert all(_equal(x, y) for x, y in zip(a, b))
    # A replay after the plan is gone still finds its tables.
    one(eager[0], eager[4])
    del plan
    fill = [torch.full((4096,), 255, dtype=torch.uint8, device="cuda")
            for _ in range(64)]
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(params[1], eager[1][1]) and len(fill) == 64


@pytest.mark.parametrize("bits", [32, 8])
def test_other_streams_and_a_plan_that_ends(bits):
    want = _small_plan(bits)
    ops.adamw_step(want[0], want[4], **HYPER)
    plan, params, state, steps, grads = _small_plan(bits)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        ops.adamw_step(plan, grads, **HYPER)
    del plan  # its tables may not go to the next allocations yet
    fill = [torch.full((512,), 255, dtype=torch.uint8, device="cuda")
            for _ in range(64)]
    torch.cuda.synchronize()
    assert len(fill) == 64
    for a, b in zip(params, want[1]):
        assert torch.equal(a, b)


def test_norms_on_streams_at_once():
    # Each with its own counters: many in flight on several streams, and beside
    # them a graph's.
    xs = [torch.randn(3_000_000 + 1000 * k, device="cuda") for k in range(4)]
    want = [ops.grad_norm(x) for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = ops.grad_norm(xs[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(20):
        for x, stream, out in zip(xs, streams, got):
            with torch.cuda.stream(stream):
                out.append(ops.grad_norm(x))
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(inside, want[0])
    for w, out in zip(want, got):
        assert all(torch.equal(w, x) for x in out)


@pytest.mark.parametrize("bits", [32, 8])
def test_no_elements_and_no_dimensions(bits):
    make = ops.adamw8_plan if bits == 8 else ops.adamw_plan
    empty = [torch.zeros(0, device="cuda"), torch.zeros(3, 0, device="cuda")]

    def state(p):
        return ops.adamw8_state(p) if bits == 8 else [torch.zeros_like(p)
                                                      for _ in range(2)]
    for params in (empty, [torch.ones((), device="cuda")] + empty):
        steps = torch.zeros(len(params), dtype=torch.int32, device="cuda")
        plan = make(params, *[list(c) for c in zip(*map(state, params))],
                    steps)
        for k in range(3):
            ops.adamw_step(plan, [None] * len(params), lr=0.5)
            ops.adamw_step(plan, [torch.ones_like(p) for p in params], lr=0.5,
                           weight_decay=0.)
            assert steps.tolist() == [k + 1] * len(params)
    # Three steps of 0.5 from 1. A code is off by an eighth at most: with 8 bits m
    # is off by 0.9 * 0.1 / 0.19 / 8 = 0.06 in the second step and by (0.06 +
    # 0.125) 0.9 * 0.19 / 0.271 = 0.12 in the third, r by 0.07 and 0.14 (half of
    # v's 0.5 * 0.266 and 0.667 * 0.43), so the steps by 0.14 and 0.3 of 0.5.
    assert float(params[0]) == pytest.approx(
        -0.5, abs=1e-5 if bits == 32 else 0.22)


def test_a_capture_before_the_first_step_is_refused():
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = AdamW([p], lr=0.5, weight_decay=0.)
    p.grad = torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    assert int(opt.state[p]["step"]) == 2
    torch.testing.assert_close(p.detach(), torch.zeros(8, device="cuda"),
                               rtol=0, atol=1e-5)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_and_a_parameter_that_comes_later(bits):
    def start():
        params = [torch.nn.Parameter(t.cuda()) for t in _tensors([70, 300, 5])]
        opt = AdamW(params, lr=1e-2, state_bits=bits, rounding_seed=3)
        for p in params[1:]:
            p.grad = torch.ones_like(p)
        opt.step()
        return params, opt

    (params, opt), (plain, opt2) = start(), start()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        if k % 2:
            for own in (params, plain):
                own[0].grad = torch.full((70,), 0.5, device="cuda")
            opt.step()
            opt2.step()
        else:
            for own in (params, plain):
                own[0].grad = None
            graph.replay()
            opt2.step()
        torch.cuda.synchronize()
        assert [int(opt.state[p]["step"]) for p in params[1:]] == [k + 2] * 2
        for p, q in zip(params, plain):
            assert torch.equal(p, q)
            x, y = opt.state.get(p, {}), opt2.state.get(q, {})
            assert set(x) == set(y) and all(_equal(x[n], y[n]) for n in x)


@pytest.mark.parametrize("sizes", [[33, 5000, 70], [2049, 2300000]])
def test_places_stand_for_tensors(sizes):
    # Two plans over parts of a list, against the plan over all of it.
    out = []
    for parts in ([range(len(sizes))], [[len(sizes) - 1],
                                        range(len(sizes) - 1)]):
        p, g = _cuda(_tensors(sizes)), _cuda(_tensors(sizes, seed=5))
        state = [_cuda(column) for column in _state8(sizes)]
        for part in parts:
            pick = lambda x: [x[i] for i in part]  # noqa: E731
            steps = torch.zeros(len(part), dtype=torch.int32, device="cuda")
            ops.adamw_step(ops.adamw8_plan(
                pick(p), *map(pick, state), steps, seed=9, places=part),
                pick(g), **HYPER)
        out.append((p, state))
    for a, b in zip(out[0][0], out[1][0]):
        assert torch.equal(a, b)
    for a, b in zip(out[0][1], out[1][1]):
        assert all(_equal(x, y) for x, y in zip(a, b))
    with pytest.raises(RuntimeError, match="places"):
        ops.adamw8_plan(p, *state, torch.zeros(
            len(sizes), dtype=torch.int32, device="cuda"), places=[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_states_replaced_before_a_capture(bits):
    p = torch.nn.Parameter(torch.ones(70, device="cuda"))
    opt = AdamW([p], lr=0.5, weight_decay=0., state_bits=bits)
    p.grad = torch.ones(70, device="cuda")
    opt.step()
    opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"].clone()
    before = p.detach().clone()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p, before) and int(opt.state[p]["step"]) == 1
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert int(opt.state[p]["step"]) == 3 + k


def test_counts_of_a_captured_step_stay():
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = AdamW([p], lr=0.5, weight_decay=0.)
    p.grad = torch.ones(8, device="cuda")
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    kept = dict(opt.state[p])  # the captured step's own, but for the counts
    at = kept.pop("step").data_ptr()
    opt.load_state_dict(opt.state_dict())
    opt.step()
    # The optimizer counts elsewhere now; that memory is nobody else's.
    assert opt.state[p]["step"].data_ptr() != at
    torch.cuda.synchronize()
    others = [torch.zeros(1, dtype=torch.int32, device="cuda")
              for _ in range(4096)]
    assert at not in {t.data_ptr() for t in others}
    graph.replay()
    torch.cuda.synchronize()
    assert int(opt.state[p]["step"]) == 2
    assert not bool(torch.stack(others).any())


def test_parameters_that_moved():
    plan, params, state, steps, grads = _small_plan(32)
    want = _small_plan(32)
    for k in range(3):
        for p in params:
            p.data = p.data.clone()
        ops.adamw_step(plan, grads, **HYPER)
        ops.adamw_step(want[0], want[4], **HYPER)
    for a, b in zip(params, want[1]):
        assert torch.equal(a, b)
    params[0].data = torch.zeros(99, device="cuda")
    with pytest.raises(RuntimeError):
        ops.adamw_step(plan, grads, **HYPER)


def test_autograd_sees_the_step():
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = AdamW([p], lr=0.1)
    p.grad = torch.ones(8, device="cuda")
    loss = (p * p).sum()
    before = p._version
    opt.step()
    assert p._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_refusals_of_the_extension():
    z = lambda n=40, d=torch.float32: torch.zeros(  # noqa: E731
        n, dtype=d, device="cuda")
    steps = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = z()
    for args in (([p], [z(41)], [z()], steps), ([p], [], [z()], steps),
                 ([p], [z().cpu()], [z()], steps),
                 ([p], [z(40, torch.bfloat16)], [z()], steps),
                 ([z(80)[::2]], [z()], [z()], steps),
                 ([z(40, torch.float64)], [z()], [z()], steps),
                 ([p], [p], [z()], steps), ([p], [z()], [z()], steps.float()),
                 ([p], [z()], [z()], steps.cpu()),
                 ([p], [z()], [z()], steps.expand(2))):
        with pytest.raises(RuntimeError):
            ops.adamw_plan(*args)
    codes, scale, *root = ops.adamw8_state(p)
    for args in (([p], [codes], [scale[:1]], *[[x] for x in root], steps),
                 ([p], [p.clone()], [scale], *[[x] for x in root], steps),
                 ([p], [codes], [scale.cpu()], *[[x] for x in root], steps),
                 ([p], [codes], [scale], [codes], [root[1]], steps)):
        with pytest.raises(RuntimeError):
            ops.adamw8_plan(*args)
    plan = ops.adamw_plan([p], [z()], [z()], steps)
    for grads in ([], [z(41)], [z().cpu()], [z(40, torch.float64)], [p],
                  [p.view(40)], [z().to_sparse()], [z(), z()]):
        with pytest.raises(RuntimeError):
            ops.adamw_step(plan, grads, lr=0.1)
    for norm in (torch.ones(()), torch.ones(2, device="cuda"),
                 torch.ones((), dtype=torch.float64, device="cuda"), p[:1]):
        with pytest.raises(RuntimeError):
            ops.adamw_step(plan, [z()], lr=0.1, norm=norm, max_norm=1.)
    for bad in ([z(3, torch.int32)], [z(), z().cpu()], [z().to_sparse()]):
        with pytest.raises(RuntimeError):
            ops.grad_norm(bad)
    assert int(steps) == 0 and not bool(p.any())
    half = z(8, torch.bfloat16)
    plan = ops.adamw_plan([half], [z(8)], [z(8)], steps)
    with pytest.raises(RuntimeError):
        ops.adamw_step(plan, [z(8)], lr=0.1)


def test_views_that_negate():
    # The imaginary part of a conjugate: its memory holds the opposite numbers.
    def minus(x):
        out = torch.complex(torch.zeros_like(x), -x).conj().imag
        assert out.is_neg() and torch.equal(out, x)
        return out

    def new():
        return [torch.ones(1, device="cuda") for _ in range(3)]
    steps = torch.zeros(1, dtype=torch.int32, device="cuda")
    for k in range(3):
        p, m, v = (minus(x) if i == k else x for i, x in enumerate(new()))
        with pytest.raises(RuntimeError, match="negates"):
            ops.adamw_plan([p], [m], [v], steps)
    p, m, v = new()
    plan = ops.adamw_plan([p], [m], [v], steps)
    five = torch.full((1,), 5., device="cuda")
    with pytest.raises(RuntimeError, match="negates"):
        ops.adamw_step(plan, [five], lr=0.1, norm=minus(five), max_norm=1.)
    # Gradients are only read: they may be.
    assert float(ops.grad_norm([minus(five)])) == 5
    ops.adamw_step(plan, [minus(five)], lr=0.1, beta1=0.5)
    assert float(m) == 3 and int(steps) == 1


def test_no_plan_is_laid_out_in_a_capture():
    plan, params, state, steps, grads = _small_plan(32)
    before = params[0].clone()
    params[0].data = params[0].data.clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            ops.adamw_step(plan, grads, **HYPER)
    torch.cuda.synchronize()
    assert torch.equal(params[0], before)


# ---------------------------------------------------------------------------- #
# Together, as training uses them


@pytest.mark.parametrize("bits", [32, 8])
def test_aggregate_norm_step(bits):
    """GAR, norm and step on the flat aggregated gradient, against the same
    calls on the CPU."""
    shapes = [(10, 3, 5, 5), (10,), (77, 13), (77,), (1,)]
    out = []
    for device in ("cpu", "cuda"):
        gen = torch.Generator().manual_seed(4)
        params = [torch.nn.Parameter(torch.randn(s, generator=gen).to(device))
                  for s in shapes]
        d = sum(p.numel() for p in params)
        opt = AdamW(params, lr=1e-2, state_bits=bits, max_norm=1.)
        for _ in range(3):
            matrix = torch.randn(8, d, generator=gen).to(device)
            flat = ops.median(matrix)
            bind_grad_views(params, flat)
            opt.step()
        out.append((params, opt))
    (a, x), (b, y) = out
    for p, q in zip(a, b):
        # A median is one of its inputs, so gradients are the same bits. The
        # norm's rounding may differ by u, and so may each step by 40 u.
        torch.testing.assert_close(p, q.cpu(), rtol=1e-6, atol=1e-6)
        if bits == 32:
            for k in ("exp_avg", "exp_avg_sq"):
                torch.testing.assert_close(x.state[p][k],
                                           y.state[q][k].cpu(),
                                           rtol=1e-5, atol=1e-8)
        assert int(y.state[q]["step"]) == 3


def _engine(args, graphs):
    exp = experiments.instantiate("mnist", ["batch-size:16"])
    return Engine(exp, "krum", WorkerGroup(5, device="cuda:0"), nbbyzwrks=1,
                  optimizer="adamw", optimizer_args=args, seed=5,
                  use_graphs=graphs, graph_warmup=2)


@pytest.mark.parametrize("args", [[], ["state-bits:8", "clip-norm:0.5"]])
def test_engine_captures_the_step(args):
    plain, captured = _engine(args, False), _engine(args, True)
    for _ in range(8):
        a, b = plain.step(), captured.step()
        assert math.isfinite(a) and math.isfinite(b)
    assert captured.use_graphs and captured._graphstep is not None \
        and captured._graphstep.ready, "graph capture did not engage"
    for p, q in zip(plain.params, captured.params):
        # Eight steps of 1e-3 whose gradients may differ in their last bits.
        torch.testing.assert_close(p, q, rtol=1e-2, atol=1e-3)
    assert int(captured.optimizer.state[captured.params[0]]["step"]) == 8


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_on_the_gpu(bits):
    one = _engine([f"state-bits:{bits}"], False)
    for _ in range(3):
        one.step()
    file = io.BytesIO()
    torch.save(one.state_dict(), file)
    file.seek(0)
    two = _engine([f"state-bits:{bits}"], False)
    two.step()
    two.load_state_dict(torch.load(file, weights_only=True,
                                   map_location="cpu"))
    for p, q in zip(one.params, two.params):
        x, y = one.optimizer.state[p], two.optimizer.state[q]
        assert all(_equal(x[k], y[k]) for k in x)
    grad = torch.randn(one.d, device="cuda")
    one.apply(grad)
    two.apply(grad)
    for p, q in zip(one.params, two.params):
        assert torch.equal(p, q)
