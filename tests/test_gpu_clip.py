"""The norm of many gradients, and the gradients clipped to it, against double precision.

Tolerances: squares and their sum are in double, the norm is rounded once to single precision (2^-24 of it, and 2^-40 for the sums); the factor is
rounded once, and so is each product: 2^-23 of a single-precision result together, 2^-8 + 2^-23 of a bfloat16 one."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(sizes, types, seed=0, size=1.0):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    return [(size * 10.0 ** (i % 5 - 4) * torch.randn(n, generator=r, device="cuda")).to(types[i % len(types)]) for i, n in enumerate(sizes)]


def norm_of(ders):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in ders))


def check(capi, ders, outs, most, run):
    want = norm_of(ders)
    factor = most / want if want > most else 1.0
    before = [g.clone() for g in ders]
    norm = run()
    assert abs(float(norm) - want) <= (2.0 ** -24 + 2.0 ** -40) * want, (float(norm), want)
    for g, y in zip(before, outs):
        if want <= most:
            assert torch.equal(g, y)
            continue
        step = 2.0 ** -23 + (2.0 ** -8 if g.dtype == torch.bfloat16 else 0.0)
        off = (y.double() - g.double() * factor).abs() - step * (g.double() * factor).abs() - 2.0 ** -149
        assert y.numel() == 0 or float(off.max()) <= 0


SIZES = [[1], [3, 1, 2], [5000], [8192, 8193, 8191], [64 * 576] * 3, [0, 7, 0, 100001, 0], [1] * 129, [17] * 500, [(i * 7919) % 3000 for i in range(300)],
         [3000001, 5, 70001], [30000000, 11]]


@pytest.mark.parametrize("types", [[torch.float32], [torch.bfloat16], [torch.bfloat16, torch.float32]])
@pytest.mark.parametrize("sizes", range(len(SIZES)))
def test_norm_and_clipping(capi, sizes, types):
    ders = make(SIZES[sizes], types, sizes)
    want = norm_of(ders)
    assert abs(float(capi.gradient_norm(ders)) - want) <= (2.0 ** -24 + 2.0 ** -40) * want
    for most in (0.25 * want, 4.0 * want, 0.0):
        outs = [torch.full_like(g, 7.0) for g in ders]
        plan = capi.GradientList(ders, outs)
        check(capi, ders, outs, most, lambda: capi.clip_gradients(plan, most))
    check(capi, ders, ders, 3.0 * want, lambda: capi.clip_gradients(ders, 3.0 * want))   # in place: as they were
    check(capi, ders, ders, 0.3 * want, lambda: capi.clip_gradients(ders, 0.3 * want))   # in place


def test_addresses_that_start_anywhere(capi):
    room = torch.randn(100003, device="cuda")
    room16 = torch.randn(100003, device="cuda").bfloat16()
    cuts = [1, 2, 1000, 9001, 9004, 50001, 100003]
    pieces = lambda t: [t[a:b] for a, b in zip(cuts, cuts[1:])]
    ders = pieces(room) + pieces(room16)
    out, out16 = torch.full_like(room, 3.0), torch.full_like(room16, 3.0)
    outs = pieces(out) + pieces(out16)
    check(capi, ders, outs, 1.0, lambda: capi.clip_gradients(capi.GradientList(ders, outs), 1.0))
    assert float(out[0]) == 3.0 and float(out16[0]) == 3.0


@pytest.mark.parametrize("size", [1e-30, 1e25])
def test_neither_overflow_nor_underflow(capi, size):
    ders = make([1000, 50000], [torch.float32], 3, size)
    outs = [torch.empty_like(g) for g in ders]
    check(capi, ders, outs, 1e-32, lambda: capi.clip_gradients(capi.GradientList(ders, outs), 1e-32))


def test_what_is_not_finite(capi):
    """An infinite norm takes all finite values to 0; one that is no number leaves them as they are"""
    ders = make([1000, 20000], [torch.float32], 4)
    ders[1][777] = math.inf
    outs = [torch.empty_like(g) for g in ders]
    norm = capi.clip_gradients(capi.GradientList(ders, outs), 1.0)
    assert float(norm) == math.inf and bool((outs[0] == 0).all()) and bool(torch.isnan(outs[1][777]))
    ders[1][5] = math.nan
    norm = capi.clip_gradients(capi.GradientList(ders, outs), 1.0)
    assert bool(torch.isnan(norm).all()) and torch.equal(outs[0], ders[0])


def test_same_bits_streams_and_graphs(capi):
    ders = make([30000, 5, 1000000, 77777], [torch.float32, torch.bfloat16], 5)
    outs = [torch.empty_like(g) for g in ders]
    plan = capi.GradientList(ders, outs)
    norm = capi.clip_gradients(plan, 0.5)
    want = [norm] + [y.clone() for y in outs]
    torch.cuda.synchronize()
    others, streams = [[torch.empty_like(g) for g in ders] for _ in range(2)], [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, o in zip(streams, others):
        with torch.cuda.stream(s):
            got.append([capi.clip_gradients(capi.GradientList(ders, o), 0.5)] + o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = capi.clip_gradients(plan, 0.5)
    second = [torch.empty_like(g) for g in ders]
    for i in range(3):
        ders[0].mul_(1.5)
        eager = capi.clip_gradients(capi.GradientList(ders, second), 0.5)
        for y in outs:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager) and all(torch.equal(a, b) for a, b in zip(outs, second)), i


@pytest.mark.parametrize("nesterov", [False, True])
def test_solver_step_with_clipping(capi, nesterov):
    """mcn_sgd_momentum_clipped is mcn_sgd_momentum with the scale that the norm gives"""
    counts = [5, 1024, 3000, 100000]
    offsets, chunks, chunk_param = capi.sgd_arena_layout(counts)
    r = torch.Generator(device="cuda")
    r.manual_seed(7)
    arena = lambda: torch.randn(chunks * capi.SGD_CHUNK, generator=r, device="cuda")
    value, state, der = arena(), arena(), arena()
    keep = torch.zeros_like(der)
    for o, n in zip(offsets, counts):
        keep[o:o + n] = 1
    der *= keep
    table = torch.from_numpy(chunk_param).cuda()
    rates = torch.tensor([[1, 1], [2, 0], [0, 0], [1, 0.5]], dtype=torch.float64, device="cuda")
    for scale, most in ((1.0, 10.0), (0.25, 1.0), (1.0, 1e9), (1.0, 0.0)):
        want = abs(scale) * float(der.double().square().sum().sqrt())
        factor = most / want if want > most else 1.0
        v1, s1, v2, s2, d = value.clone(), state.clone(), value.clone(), state.clone(), der.clone()
        norm = capi.sgd_momentum_clipped(v1, s1, d, table, rates, 0.1, 1e-4, 0.9, most, der_scale=scale, nesterov=nesterov)
        assert abs(float(norm) - want) <= (2.0 ** -24 + 2.0 ** -40) * want
        assert torch.equal(d, der)
        if factor == 1.0:
            capi.sgd_momentum(v2, s2, der, table, rates, 0.1, 1e-4, 0.9, der_scale=scale, nesterov=nesterov)
            assert torch.equal(v1, v2) and torch.equal(s1, s2)
            continue
        # state = momentum*state - (factor*der + decay*value): the factor's rounding (2^-24, and 2^-40 of the norm) and four more of magnitudes
        decay = torch.repeat_interleave(1e-4 * rates[:, 1], torch.tensor([-(-n // 1024) * 1024 for n in counts], device="cuda"))
        rate = torch.repeat_interleave(0.1 * rates[:, 0], torch.tensor([-(-n // 1024) * 1024 for n in counts], device="cuda"))
        on = (rate > 0) | (decay > 0)
        g = scale * factor * der.double()
        step = 0.9 * state.double() - g - decay * value.double()
        size = 0.9 * state.double().abs() + g.abs() + decay * value.double().abs()
        assert bool(((s1.double() - torch.where(on, step, state.double())).abs() <= 2.0 ** -21 * size + 1e-30).all())
        delta = 0.9 * step - g - decay * value.double() if nesterov else step
        moved = torch.where(on, value.double() + rate * delta, value.double())
        assert bool(((v1.double() - moved).abs() <= 2.0 ** -20 * (value.double().abs() + rate * (2 * size)) + 1e-30).all())


def test_refusals(capi):
    a, b = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")
    for bad in [lambda: capi.GradientList([a], []), lambda: capi.GradientList([a.cpu()]), lambda: capi.GradientList([a[::2]]),
                lambda: capi.GradientList([a, a]), lambda: capi.GradientList([a], [b[:5]]), lambda: capi.GradientList([a[:6], a[5:]]),
                lambda: capi.GradientList([a, b], [a, a]), lambda: capi.GradientList([a[:5], b[:5]], [b[:5], a[:5]]),
                lambda: capi.GradientList([a[:5]], [a[1:6]])]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        capi.GradientList([a.double()])
    with pytest.raises(capi.McnError) as e:
        capi.clip_gradients([a], -1.0)
    assert e.value.code == capi.ILLEGAL_ARGUMENT
    assert float(capi.gradient_norm([])) == 0.0 and float(capi.clip_gradients([], 1.0)) == 0.0
