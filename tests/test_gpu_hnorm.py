"""Heads normalised and rotated by their positions against the formulas in double precision, element by element.

Tolerances, with u = 2^-24 and h = 2^-8 for bfloat16 outputs (half a step of 2^-7).  The mean of D squares takes at most D/64 + 16 additions one
behind the other (8 channels a lane and chunk, a tree over the lanes), and the root and the quotient a rounding each: 1/sigma is off by
n = (D/64 + 16) u of itself, u_ = g x/sigma by n + 2 u.  An angle is brought to a revolution in double, rounded once as a number of half
revolutions below 1 (pi u at most) and its sine is off by 2 u: a = 8 u on cosine and sine.  A rotated channel: (n + 6 u)(|u_lo| + |u_hi|) + a (|u_lo| + |u_hi|).
Backward: du as such a channel of dzdy (a + 4 u); products with xh and their mean: (2 n + a + D/64 u + 16 u) of the magnitudes; sums over
positions and heads: a lane's share one behind the other (rows / 16 at most, in one of 2 workgroups per CU), then 32 groups, then in double."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def make(N, heads, keyHeads, D, pairs, axes, dtype, seed=0, far=0):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=r, device="cuda")
    q, k = (1.5 * normal(N, heads, D)).to(dtype), normal(N, keyHeads, D).to(dtype)
    dyq, dyk = normal(N, heads, D).to(dtype), normal(N, keyHeads, D).to(dtype)
    gq, gk = 0.5 + torch.rand(D, generator=r, device="cuda"), 0.5 + torch.rand(D, generator=r, device="cuda")
    positions = far + torch.randint(0, 1000, (N, axes), generator=r, device="cuda").double() if pairs else None
    frequencies = None
    if pairs:
        frequencies = torch.zeros(axes, pairs, dtype=torch.float64, device="cuda")
        for j in range(pairs):
            frequencies[j * axes // pairs, j] = 10000.0 ** (-j / pairs)
        frequencies[0, 0] = 1.0
    return q, k, gq, gk, dyq, dyk, positions, frequencies


class Want:
    def __init__(self, x, g, dy, positions, frequencies, eps, normalise, neighbours):
        D = x.shape[-1]
        h = 2.0 ** -8 if x.dtype == torch.bfloat16 else 0.0
        n, a = (D / 64 + 16) * U, 8 * U
        x, dy = x.double(), dy.double()
        g = torch.ones(D, dtype=torch.float64, device=x.device) if g is None else g.double()
        P = 0 if positions is None else frequencies.shape[1]
        lo = torch.arange(P, device=x.device) * (2 if neighbours else 1)
        hi = lo + (1 if neighbours else P)
        angle = (positions @ frequencies).unsqueeze(1) if P else None

        def rotated(t, sign):
            out = t.clone()
            if P:
                c, s = torch.cos(angle), sign * torch.sin(angle)
                out[..., lo], out[..., hi] = t[..., lo] * c - t[..., hi] * s, t[..., hi] * c + t[..., lo] * s
            return out

        def both(t):   # |lo| + |hi| at both channels of a pair
            out = t.abs().clone()
            if P:
                out[..., lo] = out[..., hi] = t[..., lo].abs() + t[..., hi].abs()
            return out

        r = 1.0 / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + eps) if normalise else torch.ones_like(x[..., :1])
        xh = x * r
        u = xh * g
        off = n if normalise else 0.0
        self.y, self.y_off = rotated(u, 1), (off + 6 * U + a) * both(u)
        self.y_off += h * self.y.abs()
        du = rotated(dy, -1)
        du_off = (a + 4 * U) * both(dy)
        if normalise:
            A = du * g
            product, size = (A * xh).mean(dim=-1, keepdim=True), (A * xh).abs().mean(dim=-1, keepdim=True)
            self.dx = (A - xh * product) * r
            A_off = du_off * g.abs() + 2 * U * A.abs()
            product_off = (A_off * xh.abs()).mean(dim=-1, keepdim=True) + (2 * n + 2 * U) * size
            self.dx_off = r * (A_off + xh.abs() * product_off + (2 * n + 4 * U) * (A.abs() + (xh * product).abs()))
            rows = x.shape[0] * x.shape[1]
            m = (rows / 16 + 64) * U
            self.dg = (du * xh).sum(dim=(0, 1))
            self.dg_off = (du_off * xh.abs() + (m + n + 2 * U) * (du * xh).abs()).sum(dim=(0, 1))
        else:
            self.dx, self.dx_off = du, du_off
        self.dx_off = self.dx_off + h * self.dx.abs()


def near(got, want, off, what):
    got = got.double()
    assert bool(torch.isfinite(got).all()), what + " is not finite"
    bad = (got - want).abs() - (off + 1e-30)
    assert float(bad.max()) <= 0, (what, float(bad.max()), float((got - want).abs().max()))


def check_all(capi, q, k, gq, gk, dyq, dyk, positions, frequencies, eps=1e-6, normalise=True, neighbours=False):
    how = dict(epsilon=eps, normalise=normalise, neighbours=neighbours)
    if not normalise:
        gq = gk = None
    yq, yk = capi.hnorm_forward(q, k, gq, gk, positions, frequencies, **how)
    dq, dk, dgq, dgk = capi.hnorm_backward(q, k, gq, gk, positions, frequencies, dyq, dyk, **how)
    for x, g, dy, y, dx, dg, name in ((q, gq, dyq, yq, dq, dgq, "q"), (k, gk, dyk, yk, dk, dgk, "k")):
        if x is None:
            assert y is None and dx is None and dg is None
            continue
        w = Want(x, g, dy, positions, frequencies, eps, normalise, neighbours)
        assert y.dtype == x.dtype and y.shape == x.shape
        near(y, w.y, w.y_off, "y" + name)
        near(dx, w.dx, w.dx_off, "d" + name)
        if normalise:
            near(dg, w.dg, w.dg_off, "dg" + name)
        else:
            assert dg is None
    return yq, yk, dq, dk, dgq, dgk


CASES = [  # N, heads, keyHeads, D, pairs, axes
    (1, 1, 1, 2, 1, 1), (1, 32, 8, 128, 64, 1), (16, 32, 8, 128, 64, 1), (5, 3, 1, 64, 32, 2), (33, 12, 12, 64, 32, 2), (7, 5, 5, 16, 8, 1), (100, 4, 2, 80, 40, 3),
    (64, 7, 7, 75, 24, 1), (9, 2, 1, 1, 0, 0), (9, 2, 1, 33, 16, 1), (50, 3, 3, 96, 16, 2), (50, 3, 3, 96, 13, 2), (3, 2, 2, 256, 128, 3), (4, 2, 1, 300, 150, 2),
    (4, 2, 1, 512, 256, 1), (4, 3, 2, 511, 255, 1), (6, 2, 2, 130, 65, 1), (2000, 16, 4, 128, 64, 3), (3000, 1, 1, 64, 0, 0), (1111, 3, 2, 72, 36, 2), (40, 64, 64, 32, 8, 4),
    (513, 5, 0, 64, 32, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_both_directions(capi, case, normalise, neighbours, dtype):
    N, heads, keyHeads, D, pairs, axes = CASES[case]
    q, k, gq, gk, dyq, dyk, positions, frequencies = make(N, heads, keyHeads, D, pairs, axes, dtype, case)
    if keyHeads == 0:
        k = dyk = None
    check_all(capi, q, k, gq, gk, dyq, dyk, positions, frequencies, normalise=normalise, neighbours=neighbours)
    if case % 5 == 0:   # keys alone, no multipliers
        check_all(capi, None, q, None, None, None, dyq, positions, frequencies, normalise=normalise, neighbours=neighbours)


@pytest.mark.parametrize("dtype", TYPES)
def test_far_positions(capi, dtype):
    """Position 10^6 to 10^9: the angle is as exact as near 0 (in single precision it would be off by whole radians)"""
    for far in (1000003, 123456789, 10 ** 9):
        q, k, gq, gk, dyq, dyk, positions, frequencies = make(20, 4, 2, 64, 32, 2, dtype, 1, far=far)
        check_all(capi, q, k, gq, gk, dyq, dyk, positions, frequencies)


def test_angles_of_several_axes_at_once(capi):
    """A pair may turn by all axes together, and by fractions of a position"""
    q, k, gq, gk, dyq, dyk, positions, _ = make(50, 4, 2, 64, 32, 3, torch.float32, 2)
    f = torch.randn(3, 32, dtype=torch.float64, generator=torch.Generator().manual_seed(0)).cuda()
    check_all(capi, q, k, gq, gk, dyq, dyk, positions / 7, f)


def test_the_usual_frequencies(capi):
    f = capi.axis_frequencies([4, 6, 6], 3)
    assert f.shape == (3, 16) and f.dtype == torch.float64
    want = 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    assert torch.allclose(f.sum(dim=0).cpu(), want, rtol=1e-15)
    assert bool((f[0, :4] > 0).all()) and bool((f[0, 4:] == 0).all()) and bool((f[1, 4:10] > 0).all()) and bool((f[2, :10] == 0).all())
    for bad in ([4], [4, -1]):
        with pytest.raises(ValueError):
            capi.axis_frequencies(bad, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
def test_strides_and_in_place(capi, dtype, neighbours):
    """Parts of a projection's output, heads ahead of positions, rows that start anywhere, into their own places: within the bounds, and the same
    bits where a lane holds the same channels"""
    N, heads, keyHeads, D, pairs = 77, 6, 2, 64, 32
    q, k, gq, gk, dyq, dyk, positions, frequencies = make(N, heads, keyHeads, D, pairs, 2, dtype, 3)
    how = dict(neighbours=neighbours)
    want = check_all(capi, q, k, gq, gk, dyq, dyk, positions, frequencies, **how)
    fused = torch.cat([q, k, k], dim=1)
    part = lambda t: (t[:, :heads], t[:, heads:heads + keyHeads])
    got = check_all(capi, *part(fused), gq, gk, dyq, dyk, positions, frequencies, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, dyq, dyk)]
    got = check_all(capi, turned[0], turned[1], gq, gk, turned[2], turned[3], positions, frequencies, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # into the projection's output itself, the values beside them left alone
    yq, yk = capi.hnorm_forward(*part(fused), gq, gk, positions, frequencies, out=part(fused), **how)
    assert torch.equal(yq, want[0]) and torch.equal(yk, want[1]) and torch.equal(fused[:, heads + keyHeads:], k)
    dfused = torch.cat([dyq, dyk, dyk], dim=1)
    dq, dk, _, _ = capi.hnorm_backward(q, k, gq, gk, positions, frequencies, *part(dfused), out=part(dfused), **how)
    assert torch.equal(dq, want[2]) and torch.equal(dk, want[3]) and torch.equal(dfused[:, heads + keyHeads:], dyk)

    def shifted(t):
        room = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:] = t.reshape(-1)
        return room[1:].view(t.shape)

    check_all(capi, shifted(q), shifted(k), gq, gk, shifted(dyq), shifted(dyk), positions, frequencies, **how)
    same = q[:, :1].expand(N, heads, D)      # a head read as several
    check_all(capi, same, k, gq, gk, dyq, dyk, positions, frequencies, **how)


def test_parts_repeats_streams_and_graphs(capi):
    for dtype in TYPES:
        q, k, gq, gk, dyq, dyk, positions, frequencies = make(500, 8, 2, 128, 64, 3, dtype, 4)
        full = capi.hnorm_backward(q, k, gq, gk, positions, frequencies, dyq, dyk)
        ws = capi.Workspace()
        for want in itertools.product([True, False], repeat=4):
            got = capi.hnorm_backward(q, k, gq, gk, positions, frequencies, dyq, dyk, want=want, ws=ws)
            for g, f, wanted in zip(got, full, want):
                assert (g is None) != wanted and (g is None or torch.equal(g, f))

        def step():
            return tuple(capi.hnorm_forward(q, k, gq, gk, positions, frequencies)) + tuple(
                capi.hnorm_backward(q, k, gq, gk, positions, frequencies, dyq, dyk))

        want = step()
        torch.cuda.synchronize()
        got, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        for i in range(3):
            q.copy_(torch.roll(q, 1, 0))
            eager = step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(captured, eager)), i
            for t in captured:
                t.zero_()


def test_derivatives_against_differences(capi):
    q, k, gq, gk, dyq, dyk, positions, frequencies = make(40, 3, 1, 48, 20, 2, torch.float32, 5)
    grads = capi.hnorm_backward(q, k, gq, gk, positions, frequencies, dyq, dyk)
    step = 2.0 ** -7
    for which, grad in enumerate(grads):
        args = [q, k, gq, gk]
        direction = torch.randn(args[which].shape, generator=torch.Generator(device="cuda").manual_seed(which), device="cuda")
        values = []
        for sign in (1, -1):
            moved = [t + sign * step * direction if i == which else t for i, t in enumerate(args)]
            yq, yk = capi.hnorm_forward(*moved, positions, frequencies)
            values.append((yq.double() * dyq.double()).sum() + (yk.double() * dyk.double()).sum())
        difference = float(values[0] - values[1]) / (2 * step)
        want, size = float((grad.double() * direction.double()).sum()), float((grad.double() * direction.double()).abs().sum())
        assert abs(difference - want) <= 2e-3 * size, (which, difference, want, size)


def test_values_that_are_not_finite_stay_in_their_head(capi):
    q, k, gq, gk, dyq, dyk, positions, frequencies = make(10, 4, 2, 64, 16, 1, torch.float32, 6)
    yq, yk = capi.hnorm_forward(q, k, gq, gk, positions, frequencies)
    q2 = q.clone()
    q2[3, 1, 5], q2[4, 0, 60] = math.nan, math.inf
    y2, k2 = capi.hnorm_forward(q2, k, gq, gk, positions, frequencies)
    keep = torch.ones(10, 4, dtype=torch.bool, device="cuda")
    keep[3, 1] = keep[4, 0] = False
    assert torch.equal(y2[keep], yq[keep]) and torch.equal(k2, yk)
    # channels that are not turned take nothing from a sine of zero
    y3, _ = capi.hnorm_forward(q2, None, None, None, positions, frequencies, normalise=False)
    assert torch.equal(y3[4, 0, 32:], q2[4, 0, 32:]) and bool(torch.isfinite(y3[4, 0, :32]).all())


def test_nothing_to_do_and_refusals(capi):
    q, k, gq, gk, dyq, dyk, positions, frequencies = make(6, 4, 2, 16, 8, 2, torch.float32)
    none = torch.empty(0, 4, 16, device="cuda")
    y, _ = capi.hnorm_forward(none, None)
    assert y.shape == none.shape
    dq, dk, dgq, dgk = capi.hnorm_backward(none, None, gq, None, None, None, none, None)
    assert dq.shape == none.shape and bool((dgq == 0).all()) and dgk is None
    f, b = capi.hnorm_forward, capi.hnorm_backward
    for bad in [lambda: f(None, None), lambda: f(q, k[:3]), lambda: f(q, k[:, :, :8]), lambda: f(q, k, gq[:8], gk), lambda: f(q, k, gq, gk, positions),
                lambda: f(q, k, gq, gk, positions[:3], frequencies), lambda: f(q, k, gq, gk, positions, frequencies[:1]), lambda: f(q.cpu(), k),
                lambda: f(q, k, gq, gk, normalise=False), lambda: f(q[:, :, ::2], k[:, :, ::2]), lambda: f(q, k, out=(q,)), lambda: f(q, k, out=(q[:2], k)),
                lambda: b(q, k, gq, gk, positions, frequencies, dyq, None), lambda: b(q, k, gq, gk, positions, frequencies, dyq[:2], dyk)]:
        with pytest.raises(ValueError):
            bad()
    for bad in [lambda: f(q, k.bfloat16()), lambda: f(q, k, gq.double(), gk), lambda: f(q, k, gq, gk, positions.float(), frequencies.float()),
                lambda: f(q.half(), k.half())]:
        with pytest.raises(TypeError):
            bad()
    for bad, code in [(lambda: f(q, k, gq, gk, positions, torch.zeros(2, 9, dtype=torch.float64, device="cuda")), capi.ILLEGAL_ARGUMENT),
                      (lambda: f(torch.zeros(2, 2, 513, device="cuda"), None), capi.UNSUPPORTED), (lambda: f(q, k, epsilon=-1.0), capi.ILLEGAL_ARGUMENT),
                      (lambda: f(q, None, out=(torch.zeros(1, 4, 16, device="cuda").expand(6, 4, 16), None)), capi.ILLEGAL_ARGUMENT)]:
        with pytest.raises(capi.McnError) as e:
            bad()
        assert e.value.code == code
