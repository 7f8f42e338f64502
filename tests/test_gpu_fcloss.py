"""A fully connected layer and its loss as one operator against the formulas in double precision.

Tolerances, with u = 2^-24: a product of two held values is off by 3 u of itself (the two representations and the dropped small product),
a sum of n of them by n u of the sum of magnitudes more: dz = (D + 8) u |x| |f| for a score.  Exponentials and logarithms:
2 u of the value and 2 u of the argument's size.  P = softmax - 1 at the label: |softmax| (2 dz + 64 u + 4 u max|z|), and
2^-39 as it is held; in bfloat16 2^-8 of P and of the products' results, and of the weighted x, more.  All bounds are
taken element by element."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]
SIZES = [  # (D, K, N)
    (1, 1, 1), (1, 2, 1), (3, 5, 2), (64, 64, 64), (65, 63, 33), (128, 10, 1), (31, 257, 5), (32, 33, 129), (100, 1000, 32), (2048, 1000, 32),
    (257, 4099, 70), (512, 777, 513), (1000, 3001, 300), (64, 20000, 7), (17, 70, 3001),
]


def make(D, K, N, dtype, seed=0, spread=2.0, bias=True, skipped=True, weights=True):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    x = torch.randn((N, D, 1, 1), generator=r, device="cuda").to(dtype)
    f = (torch.randn((K, D, 1, 1), generator=r, device="cuda") * spread / math.sqrt(D)).to(dtype)
    b = torch.randn(K, generator=r, device="cuda") if bias else None
    c = torch.randint(1, K + 1, (N,), generator=r, device="cuda").float()
    if skipped and N > 1:
        c[torch.rand(N, generator=r, device="cuda") < 0.2] = 0
    w = torch.rand(N, generator=r, device="cuda") + 0.5 if weights else None
    return x, f, b, c, w


class Want:
    def __init__(self, x, f, b, c, w, dzdy=1.0, normalise=True):
        N, K = x.shape[0], f.shape[0]
        bf = x.dtype == torch.bfloat16
        x, f = x.double().reshape(N, -1), f.double().reshape(K, -1)
        D = x.shape[1]
        live = c != 0
        ww = live.double() * (1.0 if w is None else w.double().repeat(N // w.numel()))
        x = torch.where((ww != 0)[:, None], x, torch.zeros_like(x))   # (whatever an image that does not count holds)
        self.counts = ww != 0                                          # (the log sums of the others are not compared)
        z = x @ f.t() + (0 if b is None else b.double())
        finite = torch.where(torch.isfinite(z), z, torch.zeros_like(z))
        dz = (D + 8) * U * (x.abs() @ f.abs().t()) + 4 * U * finite.abs()
        most = dz.amax(dim=1, keepdim=True) + 64 * U
        self.lse = torch.logsumexp(z, dim=1)
        self.lse_off = most[:, 0] + 4 * U * self.lse.abs() + 8 * U * finite.abs().amax(dim=1)
        n, at = torch.arange(N, device=z.device), torch.where(c >= 1, c - 1, torch.zeros_like(c)).long().clamp(max=K - 1)
        terms = torch.where(ww != 0, ww * (self.lse - z[n, at]), torch.zeros_like(ww))
        div = N if normalise else 1
        self.y = terms.sum() / div
        self.y_off = (ww * (2 * self.lse_off + 8 * U * (self.lse.abs() + finite[n, at].abs()))).sum() / div + U * abs(float(self.y))
        soft = torch.exp(z - self.lse[:, None])
        p = soft.clone()
        p[n, at] -= 1.0
        p = torch.where((ww != 0)[:, None], p, torch.zeros_like(p))
        p_off = soft * (2 * self.lse_off[:, None] + 2 * dz) + 4 * U * p.abs() + 2.0 ** -39
        fac = dzdy / div
        db_off = p_off
        if bf:
            p_off = p_off + 2.0 ** -8 * p.abs()
        step = 2.0 ** -8 if bf else 3 * U
        row = (fac * ww)[:, None]
        self.dx = (row * p) @ f
        self.dx_off = row.abs() * (p_off @ f.abs() + (K + 16) * U * (p.abs() @ f.abs())) + step * self.dx.abs()
        wp = (row * p).t()
        self.df = wp @ x
        extra = 2.0 ** -8 if bf and w is not None else 0.0
        self.df_off = (row * p_off).abs().t() @ x.abs() + ((N + 16) * U + extra) * (wp.abs() @ x.abs()) + step * self.df.abs() \
            + abs(fac) * 2.0 ** -39 * float((x.abs() * ww[:, None].abs()).max() if N else 0) * p.abs().sum(dim=0)[:, None]
        self.db = wp.sum(dim=1)
        self.db_off = (row * db_off).abs().sum(dim=0) + (N + 16) * U * wp.abs().sum(dim=1)


def near(got, want, off, what):
    got = got.double().reshape(want.shape)
    assert bool(torch.isfinite(got).all()), what
    bad = (got - want).abs() - (off + 1e-37)
    assert float(bad.max()) <= 0, (what, float(bad.max()), float((got - want).abs().max()))


def check(capi, x, f, b, c, w, dzdy=0.7, normalise=True):
    want = Want(x, f, b, c, w, dzdy, normalise)
    y, lse = capi.fcloss_forward(x, f, b, c, instance_weights=w, normalise=normalise)
    near(y, want.y.reshape(1), want.y_off, "y")
    near(lse[want.counts], want.lse[want.counts], want.lse_off[want.counts], "log sums")
    for sums in (lse, None):
        dx, df, db = capi.fcloss_backward(x, f, b, c, dzdy, instance_weights=w, normalise=normalise, log_sums=sums)
        assert dx.shape == x.shape and df.shape == f.shape and dx.dtype == x.dtype and df.dtype == f.dtype
        near(dx, want.dx, want.dx_off, "dzdx")
        near(df, want.df, want.df_off, "dzdf")
        near(db, want.db, want.db_off, "dzdb")
    return y, lse, dx, df, db


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_value_and_derivatives(capi, size, dtype):
    check(capi, *make(*size, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias,skipped,weights,normalise", [(False, False, False, True), (True, False, False, False), (False, True, False, True), (False, False, True, True)])
def test_options(capi, dtype, bias, skipped, weights, normalise):
    check(capi, *make(96, 333, 65, dtype, 3, bias=bias, skipped=skipped, weights=weights), normalise=normalise)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_pieces(capi, dtype):
    """More classes than one piece takes (256 MiB of P): 8192 images; and pieces of 256 classes, the last one of 1, 7, 200 classes, aligned
    and unaligned filters."""
    check(capi, *make(40, 17000, 8192, dtype, 4))
    try:
        capi.set_tunable("fcloss_piece_kib", 16)
        for size in [(64, 513, 33), (100, 775, 40), (128, 1224, 300), (64, 256, 65)]:
            check(capi, *make(*size, dtype, 5))
    finally:
        capi.set_tunable("fcloss_piece_kib", 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_does_not_count_reaches_nothing(capi, dtype):
    """Images without a label, or of weight 0, may hold anything: NaN, infinities, the largest values."""
    x, f, b, c, w = make(70, 90, 40, dtype, 5)
    c[:] = torch.randint(1, 91, (40,), device="cuda").float()
    c[3], c[7], w[9] = 0, 0, 0
    clean = check(capi, x, f, b, c, w)
    dirty = x.clone()
    dirty[3], dirty[7], dirty[9] = float("nan"), 3e38, float("inf")
    y, lse = capi.fcloss_forward(dirty, f, b, c, instance_weights=w)
    assert torch.equal(y, clean[0])
    dx, df, db = capi.fcloss_backward(dirty, f, b, c, 0.7, instance_weights=w, log_sums=lse)
    for got, want in zip((dx, df, db), clean[2:]):
        assert torch.equal(got, want)
    for n in (3, 7, 9):
        assert not dx[n].any()
    # nobody counts
    c[:] = 0
    y, _ = capi.fcloss_forward(dirty, f, b, c)
    assert float(y) == 0.0
    for t in capi.fcloss_backward(dirty, f, b, c):
        assert not t.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_classes_taken_out_and_far_scores(capi, dtype):
    """Biases of -infinity take classes out; scores of hundreds neither overflow nor lose the differences."""
    x, f, b, c, w = make(48, 130, 30, dtype, 6)
    out = torch.arange(130, device="cuda") % 3 == 1
    b[out] = float("-inf")
    c[:] = 1 + 3 * torch.randint(0, 40, (30,), device="cuda").float()
    want = Want(x, f, b, c, w, 1.0)
    y, lse = capi.fcloss_forward(x, f, b, c, instance_weights=w)
    near(y, want.y.reshape(1), want.y_off, "y")
    dx, df, db = capi.fcloss_backward(x, f, b, c, 1.0, instance_weights=w, log_sums=lse)
    assert not df[out].any() and not db[out].any()
    near(df, want.df, want.df_off, "dzdf")
    check(capi, *make(64, 200, 20, dtype, 7, spread=60.0))
    b = torch.full((130,), -3e38, device="cuda")
    b[5] = 0.0
    c[:] = 6
    y, lse = capi.fcloss_forward(x, f, b, c)
    assert bool(torch.isfinite(lse).all())


def test_magnitudes_far_apart(capi):
    """Single precision: features of 1e-20 and 1e20 per image, filters of 1e-25: the pairs' scales take it."""
    x, f, b, c, w = make(80, 64, 12, torch.float32, 8, weights=False, skipped=False)
    check(capi, x * 1e-20, f * 1e20, b, c, None)
    check(capi, x * 1e12, f * 1e-12, b, c, None)
    check(capi, x, f * 1e-25, None, c, None)
    y, lse = capi.fcloss_forward(torch.zeros_like(x), torch.zeros_like(f), None, c)
    assert abs(float(y) - math.log(64)) <= 1e-6
    check(capi, torch.zeros_like(x), f, b, c, None)


@pytest.mark.parametrize("power", [-120, -40, 60, 118])
def test_powers_of_two(capi, power):
    """Filters by 2^p and features by 2^-p: the same scores, so dzdx by 2^p and dzdf by 2^-p.  Bit for bit where the scaling of the inputs is
    exact; at 2^-120 and 2^-118 it is not (an entry below 2^-6 or 2^-8 times that is a subnormal, rounded to a multiple of 2^-149), and what
    is compared are the formulas of the rounded inputs."""
    x, f, b, c, w = make(200, 150, 40, torch.float32, seed=9)
    up, down = 2.0 ** power, 2.0 ** -power
    check(capi, x * down, f * up, b, c, w)
    if not (torch.equal(x * down * up, x) and torch.equal(f * up * down, f)):
        return
    y, sums = capi.fcloss_forward(x, f, b, c, instance_weights=w)
    dx, df, db = capi.fcloss_backward(x, f, b, c, instance_weights=w, log_sums=sums)
    y2, sums2 = capi.fcloss_forward(x * down, f * up, b, c, instance_weights=w)
    dx2, df2, db2 = capi.fcloss_backward(x * down, f * up, b, c, instance_weights=w, log_sums=sums2)
    assert torch.equal(y2, y) and torch.equal(sums2, sums) and torch.equal(db2, db)
    assert torch.equal(dx2, dx * up) and torch.equal(df2, df * down)


def test_labels_of_any_kind(capi):
    """Labels out of range go as in vl_nnloss: behind the last class to it, below 1 (but not 0) to the first."""
    x, f, b, c, _ = make(40, 30, 6, torch.float32, 9, skipped=False, weights=False)
    c[:] = torch.tensor([1.0, 30.0, 31.0, 1e12, 0.5, 2.0], device="cuda")
    same = torch.tensor([1.0, 30.0, 30.0, 30.0, 1.0, 2.0], device="cuda")
    ya, la = capi.fcloss_forward(x, f, b, c)
    yb, lb = capi.fcloss_forward(x, f, b, same)
    assert torch.equal(ya, yb)
    for p, q in zip(capi.fcloss_backward(x, f, b, c, log_sums=la), capi.fcloss_backward(x, f, b, same, log_sums=lb)):
        assert torch.equal(p, q)


def test_the_same_as_the_layers_one_by_one(capi):
    """vl_nnconv and vl_nnloss 'softmaxlog' on the scores, both in single precision: each is off by its own rounding, and twice the
    bound of the tests above holds between them."""
    D, K, N = 512, 1000, 32
    x, f, b, c, w = make(D, K, N, torch.float32, 10)
    g = capi.conv_geom((1, 1, D, N), (1, 1, D, K))
    scores = capi.conv_forward(x, f, b, g)
    lg = capi.loss_geom((1, 1, K, N))
    y0 = capi.loss_forward(scores, c, lg, instance_weights=w)
    dz = capi.loss_backward(scores, c, 1.0, lg, instance_weights=w)
    dx0, df0, db0 = capi.conv_backward(x, f, dz, g)
    want = Want(x, f, b, c, w)
    y, lse = capi.fcloss_forward(x, f, b, c, instance_weights=w)
    near(y, y0.double(), 2 * want.y_off, "y")
    dx, df, db = capi.fcloss_backward(x, f, b, c, instance_weights=w, log_sums=lse)
    near(dx, dx0.double().reshape(N, D), 2 * want.dx_off, "dzdx")
    near(df, df0.double().reshape(K, D), 2 * want.df_off, "dzdf")
    near(db, db0.double(), 2 * want.db_off, "dzdb")


@pytest.mark.parametrize("dtype", TYPES)
def test_derivatives_against_differences(capi, dtype):
    x, f, b, c, w = make(33, 70, 20, dtype, 11)

    def value(x, f, b):
        z = x.reshape(20, -1) @ f.reshape(70, -1).t() + b
        ww = (c != 0).double() * w.double()
        return float((ww * (torch.logsumexp(z, 1) - z[torch.arange(20), (c - 1).clamp(min=0).long()])).sum() / 20)

    d = capi.fcloss_backward(x, f, b, c, 1.0, instance_weights=w)
    t = 1e-5
    for k in range(3):
        args = [x.double(), f.double(), b.double()]
        v = torch.randn_like(args[k])
        plus, minus = list(args), list(args)
        plus[k], minus[k] = args[k] + t * v, args[k] - t * v
        num = (value(*plus) - value(*minus)) / (2 * t)
        terms = d[k].double() * v
        # (rounding of 2^-7 of every term at most in bfloat16; t^2 in the differences)
        assert abs(num - float(terms.sum())) <= (2.0 ** -6 if dtype == torch.bfloat16 else 1e-5) * float(terms.abs().sum()) + 1e-8


@pytest.mark.parametrize("dtype", TYPES)
def test_views_bits_streams_and_ends(capi, dtype):
    """Tensors that start anywhere give the same bits (products of one order); so do two runs, another stream, parts of the derivatives.
    Nothing is written outside of the outputs or the workspace."""
    import ctypes as C
    D, K, N = 192, 300, 50
    x, f, b, c, w = make(D, K, N, dtype, 12)
    y, lse = capi.fcloss_forward(x, f, b, c, instance_weights=w)
    d = capi.fcloss_backward(x, f, b, c, instance_weights=w, log_sums=lse)
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    xo, fo = odd(x), odd(f)
    y2, lse2 = capi.fcloss_forward(xo, fo, odd(b), odd(c), instance_weights=odd(w))
    assert torch.equal(y, y2) and torch.equal(lse, lse2)
    for p, q in zip(d, capi.fcloss_backward(xo, fo, b, c, instance_weights=w, log_sums=lse)):
        assert torch.equal(p, q)
    for want in [(True, False, False), (False, True, False), (False, False, True)]:
        got = capi.fcloss_backward(x, f, b, c, instance_weights=w, log_sums=lse, want=want)
        for k in range(3):
            assert got[k] is None if not want[k] else torch.equal(got[k], d[k])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = capi.fcloss_backward(x, f, b, c, instance_weights=w, ws=capi.Workspace())
    s.synchronize()
    for p, q in zip(d, other):
        assert torch.equal(p, q)
    # guarded outputs and workspace
    L, g = capi.lib(), capi.fcloss_geom(x, f)
    for backward in (0, 1):
        need = L.mcn_fcloss_workspace_bytes(C.byref(g), backward)
        ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
        pad = lambda t: torch.full((t.numel() + 8,), 7.0, dtype=t.dtype, device="cuda")
        outs = [pad(t) for t in ((y, lse) if not backward else d)]
        if backward:
            capi.check(L.mcn_fcloss_backward(capi.stream(), C.byref(g), *[capi.ptr(t) for t in outs], capi.ptr(lse), capi.ptr(x), capi.ptr(f), capi.ptr(b),
                                             capi.ptr(c), N, capi.ptr(w), N, 1.0, capi.ptr(ws), need))
        else:
            capi.check(L.mcn_fcloss_forward(capi.stream(), C.byref(g), *[capi.ptr(t) for t in outs], capi.ptr(x), capi.ptr(f), capi.ptr(b), capi.ptr(c), N,
                                            capi.ptr(w), N, capi.ptr(ws), need))
        torch.cuda.synchronize()
        assert bool((ws[need:] == 0x5a).all())
        for t, full in zip(outs, (y, lse) if not backward else d):
            assert torch.equal(t[:-8], full.flatten()) and bool((t[-8:] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_captured(capi, dtype):
    x, f, b, c, w = make(128, 700, 96, dtype, 13)
    ws = capi.Workspace()
    capi.fcloss_backward(x, f, b, c, instance_weights=w, ws=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, lse = capi.fcloss_forward(x, f, b, c, instance_weights=w, ws=ws)
        d = capi.fcloss_backward(x, f, b, c, instance_weights=w, log_sums=lse, ws=ws)
    for k in range(3):
        x.copy_(torch.randn_like(x.float()).to(dtype))
        graph.replay()
        torch.cuda.synchronize()
        y2, lse2 = capi.fcloss_forward(x, f, b, c, instance_weights=w)
        assert torch.equal(y, y2) and torch.equal(lse, lse2)
        for p, q in zip(d, capi.fcloss_backward(x, f, b, c, instance_weights=w, log_sums=lse2)):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_images(capi, dtype):
    x, f = torch.empty((0, 7, 1, 1), dtype=dtype, device="cuda"), torch.ones((5, 7, 1, 1), dtype=dtype, device="cuda")
    c = torch.empty(0, device="cuda")
    y, lse = capi.fcloss_forward(x, f, None, c)
    assert float(y) == 0.0 and lse.numel() == 0
    dx, df, db = capi.fcloss_backward(x, f, None, c)
    assert dx.numel() == 0 and not df.any() and not db.any()


def test_layers_of_maps(capi):
    """A fully connected layer over H x W x C maps: what vl_nnconv takes with a filter of the map's size."""
    x, f, b, c, w = make(6 * 6 * 16, 50, 9, torch.float32, 14)
    y, lse = capi.fcloss_forward(x.view(9, 16, 6, 6), f.view(50, 16, 6, 6), b, c)
    y2, _ = capi.fcloss_forward(x, f, b, c)
    assert torch.equal(y, y2)
    dx, df, db = capi.fcloss_backward(x.view(9, 16, 6, 6), f.view(50, 16, 6, 6), b, c)
    assert dx.shape == (9, 16, 6, 6) and df.shape == (50, 16, 6, 6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("slices", [1, 2, 5])
def test_every_cut_of_the_products(capi, dtype, tile, slices):
    """Each tile, and reductions in one piece and in several: odd sizes that leave part of every tile, and tiles of several rows and
    columns; a second call finds its counters as the first left them."""
    try:
        capi.set_tunable("product_tile", tile)
        capi.set_tunable("product_slices", slices)
        for size in [(130, 261, 70), (333, 515, 300), (700, 33, 1)]:
            args = make(*size, dtype, 15)
            one = check(capi, *args)
            two = check(capi, *args)
            for p, q in zip(one, two):
                assert torch.equal(p, q)
    finally:
        capi.set_tunable("product_tile", 0)
        capi.set_tunable("product_slices", 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name,value", [("product_slices", 64), ("product_tile", 100)])
def test_cuts_and_tiles_that_there_are_not(capi, dtype, name, value):
    """More slices than are made, of reductions with more stages than that, and an unknown tile."""
    try:
        capi.set_tunable(name, value)
        check(capi, *make(2600, 300, 70, dtype, 16))
        check(capi, *make(60, 70, 3000, dtype, 17))
    finally:
        capi.set_tunable(name, 0)


@pytest.mark.parametrize("D,K,N", [(64, 64, 1), (65, 130, 2), (130, 10, 3), (192, 300, 1)])
@pytest.mark.parametrize("normalise", [True, False])
def test_weights_round_nothing_twice(capi, D, K, N, normalise):
    """bfloat16 with weights: dzdf has one rounding of P to bfloat16 and one of its own: 2^-8 each.  (Want allows it a third, of the weighted
    features, which are held to 2^-16.)"""
    x, f, b, c, w = make(D, K, N, torch.bfloat16, 18, skipped=False)
    want = Want(x, f, b, c, w, 0.7, normalise)
    y, lse = capi.fcloss_forward(x, f, b, c, instance_weights=w, normalise=normalise)
    xd, fd = x.double().reshape(N, D), f.double().reshape(K, D)
    z = xd @ fd.t() + b.double()
    p = torch.softmax(z, dim=1)
    p[torch.arange(N, device="cuda"), (c - 1).long()] -= 1.0
    wp = w.double()[:, None] * p * (0.7 / (N if normalise else 1))
    # (P's own error in single precision, scores and log sums: less than 2^-14 of it here, where scores are at most 16 = 2^4: 2^4 x 64 u)
    off = (2.0 ** -8 + 2.0 ** -14 + 2.0 ** -16 + (N + 16) * U) * (wp.abs().t() @ xd.abs())
    for log_sums in (lse, None):
        for parts in ((True, True, True), (False, True, False)):
            df = capi.fcloss_backward(x, f, b, c, 0.7, instance_weights=w, normalise=normalise, log_sums=log_sums, want=parts)[1]
            near(df, want.df, off + (2.0 ** -8) * (want.df.abs() + off), "dzdf")
    assert float(z.abs().max()) <= 16
