"""The fully connected loss in single precision where magnitudes differ inside one tensor: classes that are hardly ever likely, features of very
different columns, filters and images of very different sizes.  Against the formulas in double precision, element by element.

Tolerances, with u = 2^-24: a value is held as two half-precision ones, off by 2 u of itself at most or by 2^-39 of the largest magnitude
that it shares a scale with, whichever is more; the product of two of them leaves out one of up to 4 u: 8 u of itself, and of a sum of n, n u
more.  What shares a scale: an image's features and a class's filter in the scores; in dzdf a class's P times the images' magnitudes
and, over the images, a column of the features divided by these; in dzdx an image's P times the filters' magnitudes, and a
filter.  P = softmax - 1 at the label is off by the scores' errors, twice that of the log sum, and 5 u (exponential, weight) of itself."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, FLOOR = 2.0 ** -24, 2.0 ** -39


def make(D, K, N, seed, bias=True):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    x = torch.randn((N, D, 1, 1), generator=r, device="cuda")
    f = torch.randn((K, D, 1, 1), generator=r, device="cuda") * 2 / math.sqrt(D)
    b = torch.randn(K, generator=r, device="cuda") if bias else None
    c = torch.randint(1, K + 1, (N,), generator=r, device="cuda").float()
    w = torch.rand(N, generator=r, device="cuda") + 0.5
    return x, f, b, c, w


def near(got, want, off, what):
    got = got.double().reshape(want.shape)
    assert bool(torch.isfinite(got).all()), what
    bad = (got - want).abs() - (off + 1e-40)
    worst = int(bad.argmax())
    assert float(bad.max()) <= 0, (what, worst, float(got.flatten()[worst]), float(want.flatten()[worst]), float(off.flatten()[worst]))


def check(capi, x, f, b, c, w, dzdy=0.7):
    y, lse = capi.fcloss_forward(x, f, b, c, instance_weights=w)
    got = [capi.fcloss_backward(x, f, b, c, dzdy, instance_weights=w, log_sums=s) for s in (lse, None)]
    alone = [capi.fcloss_backward(x, f, b, c, dzdy, instance_weights=w, log_sums=lse, want=k)
             for k in ((True, False, False), (False, True, False), (False, False, True))]
    for k in range(3):
        assert torch.equal(alone[k][k], got[0][k])
    N, K = x.shape[0], f.shape[0]
    x, f, w = x.double().reshape(N, -1), f.double().reshape(K, -1), w.double()
    D = x.shape[1]
    rows, cols = x.abs().amax(dim=1, keepdim=True), f.abs().amax(dim=1, keepdim=True)   # of images, of filters
    z = x @ f.t() + (0 if b is None else b.double())
    dz = (D + 8) * U * (x.abs() @ f.abs().t()) + 4 * U * z.abs() + FLOOR * (rows * f.abs().sum(dim=1) + cols.t() * x.abs().sum(dim=1, keepdim=True))
    want_lse = torch.logsumexp(z, dim=1)
    lse_off = (dz.amax(dim=1) + 64 * U) + 4 * U * want_lse.abs() + 8 * U * z.abs().amax(dim=1)
    near(lse, want_lse, lse_off, "log sums")
    n, at = torch.arange(N, device=z.device), (c - 1).long()
    want_y = (w * (want_lse - z[n, at])).sum() / N
    near(y, want_y.reshape(1), ((w * (2 * lse_off + dz[n, at] + 8 * U * (want_lse.abs() + z[n, at].abs()))).sum() / N + U * want_y.abs()).reshape(1), "y")
    soft = torch.exp(z - want_lse[:, None])
    p = soft.clone()
    p[n, at] -= 1.0
    p = w[:, None] * p
    p_off = w[:, None] * soft * (2 * lse_off[:, None] + 2 * dz) + 5 * U * p.abs()
    p_off[n, at] += 2 * U * w   # (the label's: a difference from 1)
    fac = dzdy / N
    # dzdf: P by the images' magnitudes, features over them
    px, xx = p * rows, x / rows
    df = fac * (p.t() @ x)
    df_off = fac * (p_off.t() @ x.abs() + (N + 8) * U * (p.abs().t() @ x.abs())
                    + 4 * FLOOR * (px.abs().amax(dim=0)[:, None] * xx.abs().sum(dim=0) + xx.abs().amax(dim=0) * px.abs().sum(dim=0)[:, None])) + 3 * U * df.abs()
    pf, ff = p * cols.t(), f / cols
    dx = fac * (p @ f)
    dx_off = fac * (p_off @ f.abs() + (K + 8) * U * (p.abs() @ f.abs())
                    + 4 * FLOOR * (pf.abs().amax(dim=1, keepdim=True) * ff.abs().sum(dim=0) + pf.abs().sum(dim=1, keepdim=True))) + 3 * U * dx.abs()
    db = fac * p.sum(dim=0)
    db_off = fac * (p_off.sum(dim=0) + (N + 8) * U * p.abs().sum(dim=0))
    for have in got:
        near(have[2], db, db_off, "dzdb")
        near(have[1], df, df_off, "dzdf")
        near(have[0], dx, dx_off, "dzdx")


@pytest.mark.parametrize("D,K,N", [(96, 2000, 200), (40, 300, 7), (64, 513, 700)])
def test_classes_that_are_hardly_likely(capi, D, K, N):
    """Classes that no image has, with biases of -12 to -60: their filters' derivatives are as exact, each by itself, as the others'."""
    x, f, b, c, w = make(D, K, N, 1)
    rare = torch.arange(K, device="cuda") % 10 == 3
    b[rare] = -torch.linspace(12, 60, int(rare.sum()), device="cuda")
    c[:] = torch.where(rare[(c - 1).long()], c + 1, c)
    c.clamp_(max=float(K))
    check(capi, x, f, b, c, w)


@pytest.mark.parametrize("D,K,N", [(96, 700, 200), (40, 300, 7), (1100, 64, 130)])
@pytest.mark.parametrize("spread", [5, 8])
def test_features_of_very_different_columns(capi, D, K, N, spread):
    x, f, b, c, w = make(D, K, N, 2)
    check(capi, x * torch.logspace(-spread, 0, D, device="cuda")[None, :, None, None], f, b, c, w)


@pytest.mark.parametrize("D,K,N", [(96, 700, 200), (40, 300, 7), (257, 4099, 33)])
@pytest.mark.parametrize("spread", [5, 8, 30])
def test_filters_of_very_different_sizes(capi, D, K, N, spread):
    x, f, b, c, w = make(D, K, N, 3)
    check(capi, x, f * torch.logspace(-spread, 0, K, device="cuda")[:, None, None, None], b, c, w)


@pytest.mark.parametrize("D,K,N", [(96, 700, 200), (40, 300, 7)])
@pytest.mark.parametrize("spread", [5, 12, 30])
def test_images_of_very_different_sizes(capi, D, K, N, spread):
    x, f, b, c, w = make(D, K, N, 4)
    check(capi, x * torch.logspace(-spread, 0, N, device="cuda")[torch.randperm(N, device="cuda")][:, None, None, None], f, b, c, w)


def test_all_of_it_at_once_and_in_pieces(capi):
    """Every kind together, over one piece of the classes and over several, the last of them small."""
    D, K, N = 130, 1100, 150
    x, f, b, c, w = make(D, K, N, 5)
    x = x * torch.logspace(-3, 0, N, device="cuda")[torch.randperm(N, device="cuda")][:, None, None, None] * torch.logspace(-4, 0, D, device="cuda")[None, :, None, None]
    f = f * torch.logspace(-6, 0, K, device="cuda")[torch.randperm(K, device="cuda")][:, None, None, None]
    b[::7] = -30.0
    check(capi, x, f, b, c, w)
    try:
        capi.set_tunable("fcloss_piece_kib", 16)
        check(capi, x, f, b, c, w)
    finally:
        capi.set_tunable("fcloss_piece_kib", 0)


def test_single_entries_far_from_all_others(capi):
    """One feature, one filter value, one image and one class of their own size: nothing else may lose by it."""
    D, K, N = 70, 200, 90
    x, f, b, c, w = make(D, K, N, 6)
    x[:, 3] *= 1e-7
    x[11] *= 1e-6
    f[5] *= 1e-9
    f[17, 2] = 3e4
    x[:, 2] *= 1e-5
    check(capi, x, f, b, c, w)
