"""Layer normalisation against its formulas in double precision.

Tolerances, with u = 2^-24 (half a step of single precision): a sum of C values takes at most n = C/256 + 64 additions one behind the
other (16 values a thread and a tree over the threads, or C/256 values and a tree), so the mean is off by n u max|x| and
sigma by n u of itself; xh = (x - mu)/sigma by e = n u (max|x|/sigma + |xh|).  Everything else follows from that, and an
output in bfloat16 is off by 2^-8 of itself more."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [  # (H, W, C, N)
    (1, 1, 1, 5), (1, 1, 2, 1), (1, 1, 7, 100), (1, 1, 16, 33), (1, 1, 64, 130), (1, 1, 65, 9), (1, 1, 257, 70), (1, 1, 1000, 32), (1, 1, 1024, 17),
    (1, 1, 1023, 2100), (1, 1, 2048, 32), (1, 1, 2501, 9), (1, 1, 4096, 300), (1, 1, 5000, 11), (1, 1, 8192, 7), (1, 1, 9999, 3), (1, 1, 16384, 2),
    (1, 1, 16385, 3), (1, 1, 40000, 2),
    (2, 1, 3, 4), (5, 7, 64, 3), (7, 7, 65, 2), (3, 1, 130, 40), (14, 14, 256, 2), (56, 56, 256, 1), (9, 9, 512, 2), (3, 5, 513, 2), (4, 4, 1500, 1), (1, 63, 8, 70), (5, 3, 300, 7), (3, 3, 1024, 2), (2, 9, 700, 33), (7, 1, 1025, 2),
]
TYPES = [torch.float32, torch.bfloat16]


def make(shape, dtype, seed=0):
    H, W, C, N = shape
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    x = torch.randn((N, C, W, H), generator=r, device="cuda") * 1.5 + torch.randn((1, C, 1, 1), generator=r, device="cuda")
    dy = torch.randn((N, C, W, H), generator=r, device="cuda")
    g = torch.rand(C, generator=r, device="cuda") + 0.5
    b = torch.randn(C, generator=r, device="cuda")
    return x.to(dtype), g, b, dy.to(dtype)


class Want:
    """Formulas and bounds, in double, rows of channels."""

    def __init__(self, x, g, b, dy, eps, moments=None):
        self.shape = x.shape
        N, C, W, H = x.shape
        rows = lambda t: t.double().permute(0, 2, 3, 1).reshape(-1, C)
        x, dy = rows(x), rows(dy)
        g = torch.ones(C, dtype=torch.float64, device=x.device) if g is None else g.double()
        b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
        if moments is None:
            mu = x.mean(dim=1, keepdim=True)
            sigma = torch.sqrt(((x - mu) ** 2).mean(dim=1, keepdim=True) + eps)
        else:
            mu, sigma = moments.double().reshape(2, -1, 1)
        n = (C / 256 + 64) * U
        xh = (x - mu) / sigma
        most = x.abs().amax(dim=1, keepdim=True)
        e = n * (most / sigma + xh.abs())
        self.mu, self.sigma = mu, sigma
        self.mu_off, self.sigma_off = n * most, n * (sigma + most * most / sigma * n)
        self.y, self.y_off = xh * g + b, e * g.abs() + 2 * U * (xh * g).abs() + U * b.abs()
        a = dy * g
        A, X, E = a.abs().amax(dim=1, keepdim=True), xh.abs().amax(dim=1, keepdim=True), e.amax(dim=1, keepdim=True)
        s1, s2 = a.mean(dim=1, keepdim=True), (a * xh).mean(dim=1, keepdim=True)
        self.dx = (a - s1 - xh * s2) / sigma
        self.dx_off = (4 * n * (A + xh.abs() * A * X) + (xh.abs() * E + e * X) * A) / sigma
        # a sum over the pixels: a thread's share, then 64 lanes, 16 wavefronts and 256 workgroups
        m = (x.shape[0] / 256 + 32) * U
        self.dg, self.dg_off = (dy * xh).sum(dim=0), m * (dy * xh).abs().sum(dim=0) + (dy.abs() * e).sum(dim=0)
        self.db, self.db_off = dy.sum(dim=0), m * dy.abs().sum(dim=0)

    def back(self, t):
        N, C, W, H = self.shape
        return t.reshape(N, W, H, C).permute(0, 3, 1, 2)


def near(got, want, off, what=""):
    got = got.double()
    step = 2.0 ** -8 if got is not None and what.endswith("bf16") else 0.0
    bad = (got - want).abs() - (off + step * want.abs() + 1e-30)
    assert bool(torch.isfinite(got).all()) and float(bad.max()) <= 0, (what, float(bad.max()), float((got - want).abs().max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_both_directions(capi, shape, dtype):
    x, g, b, dy = make(shape, dtype)
    eps = 1e-5
    w = Want(x, g, b, dy, eps)
    tag = " bf16" if dtype == torch.bfloat16 else ""
    y, mom = capi.lnorm_forward(x, g, b, eps)
    assert y.dtype == dtype and mom.shape == (2,) + (x.shape[0], x.shape[2], x.shape[3])
    near(mom[0].reshape(-1, 1), w.mu, w.mu_off, "mu")
    near(mom[1].reshape(-1, 1), w.sigma, w.sigma_off, "sigma")
    near(y, w.back(w.y), w.back(w.y_off), "y" + tag)
    for moments in (mom, None):
        dx, dg, db = capi.lnorm_backward(x, g, dy, eps, moments=moments)
        near(dx, w.back(w.dx), w.back(w.dx_off), "dx" + tag)
        near(dg, w.dg, w.dg_off, "dg")
        near(db, w.db, w.db_off, "db")


@pytest.mark.parametrize("shape", [(1, 1, 100, 7), (1, 1, 20000, 3), (3, 3, 40, 5), (2, 2, 700, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_no_affine_given_moments_and_parts_of_the_derivatives(capi, shape, dtype):
    x, g, b, dy = make(shape, dtype, 1)
    H, W, C, N = shape
    tag = " bf16" if dtype == torch.bfloat16 else ""
    w = Want(x, None, None, dy, 1e-3)
    y, mom = capi.lnorm_forward(x, None, None, 1e-3)
    near(y, w.back(w.y), w.back(w.y_off), "y" + tag)
    dx, dg, db = capi.lnorm_backward(x, None, dy, 1e-3)
    near(dx, w.back(w.dx), w.back(w.dx_off), "dx" + tag)
    # only what is asked for, the same bits
    for want in [(True, False, False), (False, True, True), (False, False, True), (False, True, False)]:
        got = capi.lnorm_backward(x, None, dy, 1e-3, want=want)
        for k, full in enumerate((dx, dg, db)):
            assert (got[k] is None) == (not want[k])
            if want[k]:
                assert torch.equal(got[k], full)
    # moments of the caller's
    given = torch.stack([torch.full((N, W, H), 0.25, device="cuda"), torch.full((N, W, H), 2.0, device="cuda")])
    w = Want(x, g, b, dy, 0.0, given)
    y, same = capi.lnorm_forward(x, g, b, 0.0, moments=given)
    assert same is given
    near(y, w.back(w.y), w.back(w.y_off), "y" + tag)
    dx, dg, db = capi.lnorm_backward(x, g, dy, 0.0, moments=given)
    near(dx, w.back(w.dx), w.back(w.dx_off), "dx" + tag)
    near(dg, w.dg, w.dg_off, "dg")


def test_hard_rows(capi):
    """A constant row has variance 0: y = b, and the derivative is finite; large offsets cancel in the squares about the mean; a row
    with a NaN or an infinity does not touch its neighbours."""
    C = 300
    x = torch.zeros((4, C, 1, 1), device="cuda")
    x[0] = 3.5
    x[1] = 1e4 + torch.randn((C, 1, 1), device="cuda", generator=None)
    x[2] = 1e-20 * torch.randn((C, 1, 1), device="cuda")
    x[3] = torch.randn((C, 1, 1), device="cuda")
    g, b = torch.ones(C, device="cuda"), torch.full((C,), 0.5, device="cuda")
    dy = torch.randn_like(x)
    w = Want(x, g, b, dy, 1e-5)
    y, mom = capi.lnorm_forward(x, g, b, 1e-5)
    near(y, w.back(w.y), w.back(w.y_off), "y")
    assert torch.equal(y[0].flatten(), b)
    dx, dg, db = capi.lnorm_backward(x, g, dy, 1e-5, moments=mom)
    near(dx, w.back(w.dx), w.back(w.dx_off), "dx")
    bad = x.clone()
    bad[2, 7], bad[0, 3] = float("nan"), float("inf")
    y2, _ = capi.lnorm_forward(bad, g, b, 1e-5)
    assert torch.equal(y2[1], y[1]) and torch.equal(y2[3], y[3]) and bool(torch.isnan(y2[2]).all())


@pytest.mark.parametrize("shape", [(1, 1, 129, 50), (3, 3, 33, 9), (1, 1, 17000, 3)])
def test_derivative_against_differences(capi, shape):
    """d/dt of sum(c .* y(x + t v)) in double against the kernel's derivatives."""
    x, g, b, dy = make(shape, torch.float32, 3)
    eps = 1e-5

    def f(x, g, b):
        x = x.double()
        mu = x.mean(dim=1, keepdim=True)
        s = torch.sqrt(((x - mu) ** 2).mean(dim=1, keepdim=True) + eps)
        return float(((x - mu) / s * g.double().view(1, -1, 1, 1) + b.double().view(1, -1, 1, 1)).mul(dy.double()).sum())

    dx, dg, db = capi.lnorm_backward(x, g, dy, eps)
    t = 1e-5
    for which, d in enumerate((dx, dg, db)):
        args = [x.double(), g.double(), b.double()]
        v = torch.randn_like(args[which])
        plus, minus = list(args), list(args)
        plus[which], minus[which] = args[which] + t * v, args[which] - t * v
        num = (f(*plus) - f(*minus)) / (2 * t)
        ana = float((d.double() * v).sum())
        # (central differences: t^2 of the third derivative and 2^-53/t of the value; the kernel: 1e-5 of the terms)
        assert abs(num - ana) <= 1e-4 * float((d.double() * v).abs().sum() + 1.0), (which, num, ana)


def test_views_streams_and_bits(capi):
    """Rows that start anywhere take the same values as aligned ones to rounding; two runs and another stream give the same bits; outputs end
    where they should."""
    L = capi.lib()
    for C, N, dtype in [(1024, 33, torch.float32), (96, 50, torch.bfloat16), (1001, 20, torch.bfloat16)]:
        x, g, b, dy = make((1, 1, C, N), dtype, 5)
        w = Want(x, g, b, dy, 1e-5)
        tag = " bf16" if dtype == torch.bfloat16 else ""
        odd = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(x).copy_(x)
        guard = torch.full((x.numel() + 66,), 7.0, dtype=dtype, device="cuda")
        out = guard[1:1 + x.numel()]
        capi.check(L.mcn_lnorm_forward(capi.stream(), capi.data_type(x), capi.ptr(out), None, capi.ptr(odd), capi.ptr(g), capi.ptr(b), 1, 1, C, N, 1e-5, 0))
        near(out.view_as(x), w.back(w.y), w.back(w.y_off), "y" + tag)
        assert float(guard[0]) == 7.0 and bool((guard[1 + x.numel():] == 7.0).all())
        first = capi.lnorm_backward(x, g, dy)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            second = capi.lnorm_backward(x, g, dy, ws=capi.Workspace())
        s.synchronize()
        for p, q in zip(first, second):
            assert torch.equal(p, q)


def test_captured(capi):
    x, g, b, dy = make((1, 1, 700, 333), torch.float32, 6)
    ws = capi.Workspace()
    eager = capi.lnorm_backward(x, g, dy, ws=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mom = capi.lnorm_forward(x, g, b)
        got = capi.lnorm_backward(x, g, dy, moments=mom, ws=ws)
    for k in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        want_y, want_mom = capi.lnorm_forward(x, g, b)
        want = capi.lnorm_backward(x, g, dy, moments=want_mom)
        assert torch.equal(y, want_y)
        for p, q in zip(got, want):
            assert torch.equal(p, q)


def test_no_pixels(capi):
    x = torch.empty((0, 5, 1, 1), device="cuda")
    g = torch.ones(5, device="cuda")
    y, _ = capi.lnorm_forward(x, g, None)
    assert y.shape == x.shape
    dx, dg, db = capi.lnorm_backward(x, g, x)
    assert not dg.any() and not db.any()


def test_convert(capi):
    for n in (1, 3, 4, 1023, 100001):
        x = torch.randn(n, device="cuda") * 3
        x[0] = float("inf")
        h = capi.convert(x, torch.bfloat16)
        assert torch.equal(h, x.to(torch.bfloat16)) and torch.equal(capi.convert(h, torch.float32), h.float())
        assert torch.equal(capi.convert(h[1:], torch.float32), h[1:].float()) if n > 1 else True


@pytest.mark.parametrize("shape", [(1, 1, 2, (1 << 28) + 3), (2, 2, 2, (1 << 26) + 1)])
def test_more_threads_than_a_dimension_of_a_grid_has(capi, shape):
    """2^28 pixels of two channels, sixteen threads to a pixel."""
    H, W, C, N = shape
    x = torch.empty((N, C, W, H), dtype=torch.bfloat16, device="cuda").normal_()
    g, b = torch.tensor([0.5, 2.0], device="cuda"), torch.tensor([1.0, -1.0], device="cuda")
    y, mom = capi.lnorm_forward(x, g, b)
    at = torch.cat([torch.arange(1000), torch.arange(N - 1000, N), torch.randint(0, N, (100000,))]).cuda()
    want = Want(x[at], g, b, x[at], 1e-5)
    near(y[at], want.back(want.y), want.back(want.y_off), "bf16")
    near(mom[0, at].reshape(-1, 1), want.mu, want.mu_off, "mu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 1, 20000, 3), (7, 7, 2048, 2), (1, 3, 16385, 1), (1, 1, 20000, 3)])
def test_sums_of_many_channels(capi, shape, dtype):
    """More channels than registers hold: sums of equal values, whose roundings all go one way.  The bounds above, which count C/256 + 64 additions."""
    H, W, C, N = shape
    x, g, b, dy = make(shape, dtype, 7)
    flat = torch.linspace(0.1, 0.9, N * W * H, device="cuda").view(N, 1, W, H)
    x = (x * 0 + flat).to(dtype)
    w = Want(x, g, b, dy, 1e-5)
    tag = " bf16" if dtype == torch.bfloat16 else ""
    y, mom = capi.lnorm_forward(x, g, b, 1e-5)
    near(mom[0].reshape(-1, 1), w.mu, w.mu_off, "mu")
    near(mom[1].reshape(-1, 1), w.sigma, w.sigma_off, "sigma")
    near(y, w.back(w.y), w.back(w.y_off), "y" + tag)
    dy = (dy * 0 + flat).to(dtype)
    w = Want(x, g, b, dy, 1e-5)
    for moments in (mom, None):
        dx, dg, db = capi.lnorm_backward(x, g, dy, 1e-5, moments=moments)
        near(dx, w.back(w.dx), w.back(w.dx_off), "dx" + tag)
        near(dg, w.dg, w.dg_off, "dg")
        near(db, w.db, w.db_off, "db")


def test_as_many_channels_as_are_taken(capi):
    """2^24 channels of two pixels: more workgroups for the sums over pixels than one dimension of a grid has threads for."""
    shape = (2, 1, 1 << 24, 1)
    x, g, b, dy = make(shape, torch.float32, 8)
    y, mom = capi.lnorm_forward(x, g, b, 1e-5)
    dx, dg, db = capi.lnorm_backward(x, g, dy, 1e-5, moments=mom)
    w = Want(x, g, b, dy, 1e-5)
    near(mom[0].reshape(-1, 1), w.mu, w.mu_off, "mu")
    near(mom[1].reshape(-1, 1), w.sigma, w.sigma_off, "sigma")
    near(y, w.back(w.y), w.back(w.y_off), "y")
    near(dx, w.back(w.dx), w.back(w.dx_off), "dx")
    near(dg, w.dg, w.dg_off, "dg")
    near(db, w.db, w.db_off, "db")
