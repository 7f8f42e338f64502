"""Orthogonalised updates against the same products in double precision, and against the singular value decomposition.

Tolerance, with u = 2^-24, in Frobenius norms: every step multiplies an error that is there by at most 3.4445 (the largest slope of
p(s) = a s + b s^3 + c s^5 on [0, 1.22]) and adds its own: of A = X X', B = b A + c A^2 and X <- a X + B X, each a sum of n products
whose 3 n/16 additions (three small products, sixteen indices an instruction) round independently: 4 (sqrt(3 n/16) + 3) u of
|x_i| |x_j| at four deviations, which in norms is F(left) F(right)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
A, B, C = 3.4445, -4.7750, 2.0315


def reference(g, steps):
    """(result, bound in the Frobenius norm) of one matrix"""
    x = g.double()
    norm = torch.linalg.norm(x)
    if float(norm) == 0:
        return x, 0.0
    x = x / norm
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    m, n = x.shape
    gamma = lambda k: 4 * (math.sqrt(3 * k / 16) + 3) * U
    off = 2 * U
    for _ in range(steps):
        a = x @ x.t()
        b = B * a + C * (a @ a)
        F, s = float(torch.linalg.norm(x)), float(torch.linalg.matrix_norm(x, 2))
        Fa, Fb = float(torch.linalg.norm(a)), float(torch.linalg.norm(b))
        da = gamma(n) * F * F
        db = abs(B) * da + C * (2 * s * s * da + gamma(m) * Fa * Fa) + 3 * U * Fb
        off = 3.4445 * off + s * db + gamma(m) * Fb * F + 4 * U * A * F
        x = A * x + b @ x
    return (x.t() if tall else x), off


def check(capi, g, steps=5):
    y = capi.orthogonalise(g, steps=steps)
    assert y.shape == g.shape and bool(torch.isfinite(y).all())
    K = g.shape[1]
    for one, got in zip(g.reshape(g.shape[0], K, -1), y.reshape(g.shape[0], K, -1)):
        want, off = reference(one, steps)
        away = float(torch.linalg.norm(got.double() - want))
        assert away <= off, (tuple(g.shape), away, off)
    return y


SIZES = [(1, 1, 1), (2, 1, 7), (1, 5, 1), (3, 2, 2), (2, 31, 33), (1, 32, 32), (2, 64, 576), (3, 65, 64), (1, 64, 147), (2, 100, 257), (1, 257, 100), (1, 129, 4000),
         (1, 1000, 130), (1, 300, 300), (1, 512, 1024), (5, 16, 9), (1, 777, 1025)]


@pytest.mark.parametrize("count,K,D", SIZES)
def test_random_matrices(capi, count, K, D):
    r = torch.Generator(device="cuda")
    r.manual_seed(K * D)
    check(capi, torch.randn((count, K, D), generator=r, device="cuda") * 1e-3)


@pytest.mark.parametrize("count,K,D", [(1, 64, 2000), (1, 2001, 63), (3, 9, 900), (2, 33, 1023), (1, 120, 120), (2, 99, 130), (130, 90, 66), (300, 70, 71)])
def test_one_tile_of_products(capi, count, K, D):
    """Shapes whose X X' is one tile, also with its reduction cut into slices and with more matrices than the chip has units."""
    r = torch.Generator(device="cuda")
    r.manual_seed(K + D)
    g = torch.randn((count, K, D), generator=r, device="cuda")
    y = capi.orthogonalise(g)
    assert bool(torch.isfinite(y).all())
    for k in sorted({0, count // 2, count - 1}):
        want, off = reference(g[k], 5)
        assert float(torch.linalg.norm(y[k].double() - want)) <= off
    assert torch.equal(capi.orthogonalise(g), y)


@pytest.mark.parametrize("K,D", [(64, 200), (200, 64), (130, 130)])
def test_few_strong_directions(capi, K, D):
    r = torch.Generator(device="cuda")
    r.manual_seed(3)
    g = torch.randn((K, 4), generator=r, device="cuda") @ torch.randn((4, D), generator=r, device="cuda")
    check(capi, g[None])                                       # rank 4: the rest stays (nearly) zero
    check(capi, (g + 0.02 * torch.randn((K, D), generator=r, device="cuda"))[None])


def test_singular_values(capi):
    """From the decomposition: U p(p(...p(S/|S|))) V', and every value from 1/200 of the norm on ends within [0.68, 1.21]."""
    r = torch.Generator(device="cuda")
    r.manual_seed(4)
    g = torch.randn((1, 48, 300), generator=r, device="cuda")
    y = capi.orthogonalise(g)[0].double().cpu()
    u, s, v = torch.linalg.svd(g[0].double().cpu(), full_matrices=False)
    p = s / torch.linalg.norm(s)
    for _ in range(5):
        p = A * p + B * p ** 3 + C * p ** 5
    _, off = reference(g[0], 5)
    assert float(torch.linalg.norm(y - (u * p) @ v)) <= off
    got = torch.linalg.svdvals(y)
    assert float(got.min()) >= 0.68 and float(got.max()) <= 1.21


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-10, 1e10, 1e36])
def test_any_magnitude(capi, scale):
    """Only the direction counts; squares that leave single precision are no matter."""
    r = torch.Generator(device="cuda")
    r.manual_seed(5)
    check(capi, torch.randn((1, 40, 90), generator=r, device="cuda") * scale)


def test_zero_and_not_finite(capi):
    g = torch.randn((4, 20, 50), device="cuda")
    g[1] = 0
    clean = capi.orthogonalise(g)
    assert not clean[1].any()
    g[2, 3, 4], g[3, 0, 0] = float("nan"), float("inf")
    y = capi.orthogonalise(g)
    assert torch.equal(y[0], clean[0]) and not y[1].any() and bool(torch.isnan(y[2]).any()) and bool(torch.isnan(y[3]).any())
    one = torch.zeros((1, 33, 40), device="cuda")
    one[0, 5, 6] = -2.0                                          # one entry: a singular value of 1
    p = 1.0
    for _ in range(5):
        p = A * p + B * p ** 3 + C * p ** 5
    y = capi.orthogonalise(one)
    assert abs(float(y[0, 5, 6]) + p) <= 1e-5 and int((y != 0).sum()) == 1


@pytest.mark.parametrize("steps", [0, 1, 2, 8])
def test_steps(capi, steps):
    r = torch.Generator(device="cuda")
    r.manual_seed(6)
    for K, D in [(40, 130), (130, 40)]:
        check(capi, torch.randn((2, K, D), generator=r, device="cuda"), steps)


def test_views_bits_streams_and_ends(capi):
    L = capi.lib()
    for K, D in [(64, 200), (200, 64), (70, 70)]:
        g = torch.randn((2, K, D), device="cuda")
        y = capi.orthogonalise(g)
        odd = torch.empty(g.numel() + 1, device="cuda")[1:].view_as(g).copy_(g)
        need = L.mcn_orthogonalise_workspace_bytes(K, D, 2)
        ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
        out = torch.full((g.numel() + 9,), 7.0, device="cuda")
        capi.check(L.mcn_orthogonalise(capi.stream(), capi.ptr(out[1:]), capi.ptr(odd), K, D, 2, 5, capi.ptr(ws), need))
        torch.cuda.synchronize()
        assert torch.equal(out[1:-8].view_as(g), y) and float(out[0]) == 7.0 and bool((out[-8:] == 7.0).all()) and bool((ws[need:] == 0x5a).all())
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            z = capi.orthogonalise(g, ws=capi.Workspace())
        s.synchronize()
        assert torch.equal(z, y)
        # a bank of its own gives the bits that it gives among others
        assert torch.equal(capi.orthogonalise(g[1:].contiguous())[0], y[1])


def test_captured(capi):
    g = torch.randn((3, 64, 150), device="cuda")
    ws = capi.Workspace()
    capi.orthogonalise(g, ws=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = capi.orthogonalise(g, ws=ws)
    for k in range(3):
        g.copy_(torch.randn_like(g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, capi.orthogonalise(g))


def test_empty(capi):
    assert capi.orthogonalise(torch.empty((0, 4, 4), device="cuda")).numel() == 0


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("slices", [1, 2, 5])
def test_every_cut_of_the_products(capi, tile, slices):
    try:
        capi.set_tunable("product_tile", tile)
        capi.set_tunable("product_slices", slices)
        capi.set_tunable("ortho_no_narrow", 1)
        r = torch.Generator(device="cuda")
        r.manual_seed(7)
        for count, K, D in [(2, 70, 333), (1, 515, 300), (1, 290, 290), (3, 33, 40)]:
            g = torch.randn((count, K, D), generator=r, device="cuda")
            assert torch.equal(check(capi, g), check(capi, g))
    finally:
        capi.set_tunable("product_tile", 0)
        capi.set_tunable("product_slices", 0)
        capi.set_tunable("ortho_no_narrow", 0)


@pytest.mark.parametrize("count,K,D", [(1, 1, 1), (2, 64, 576), (2, 576, 64), (1, 63, 575), (1, 65, 64), (1, 33, 1), (1, 1, 576), (3, 31, 129), (1, 64, 577), (70, 8, 24),
                                       (1, 576, 33), (1, 64, 64)])
def test_narrow_matrices_in_one_launch(capi, count, K, D):
    """Up to 64 x 576 either way: all steps in one launch, within the same bound as the products launch by launch."""
    r = torch.Generator(device="cuda")
    r.manual_seed(8)
    g = torch.randn((count, K, D), generator=r, device="cuda")
    for steps in (1, 5):
        check(capi, g, steps)
        try:
            capi.set_tunable("ortho_no_narrow", 1)
            check(capi, g, steps)
        finally:
            capi.set_tunable("ortho_no_narrow", 0)
