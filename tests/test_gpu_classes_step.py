"""The operators for classifiers with many classes as they are used together: features -> layer normalisation -> fully connected layer and
loss -> their gradients -> orthogonalised update of the bank.  Against the same step in double precision (values), against
differences of the loss (gradients), through the front-end, and captured into a graph and replayed."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS, MOMENTUM, RATE = 1e-5, 0.9, 0.02


def make(N, C, K, seed=0):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=r, device="cuda")
    x = n(N, C, 1, 1) * 2 + 0.5
    p = dict(g=torch.rand(C, generator=r, device="cuda") + 0.5, b=n(C) * 0.1, f=n(K, C, 1, 1) / C ** 0.5, fb=n(K) * 0.1)
    c = torch.randint(0, K + 1, (N,), generator=r, device="cuda").float()   # (zeros: images that do not count)
    w = torch.rand(N, generator=r, device="cuda") + 0.5
    m = n(1, K, C) * 1e-3
    return x, p, c, w, m


def step(capi, x, p, c, w, m):
    """One training step's gradients and the bank after its update."""
    y, moments = capi.lnorm_forward(x, p["g"], p["b"], EPS)
    loss, sums = capi.fcloss_forward(y, p["f"], p["fb"], c, instance_weights=w)
    dy, df, dfb = capi.fcloss_backward(y, p["f"], p["fb"], c, 1.0, instance_weights=w, log_sums=sums)
    dx, dg, db = capi.lnorm_backward(x, p["g"], dy, EPS, moments=moments)
    momentum = capi.taccum(MOMENTUM, m, 1.0, df.reshape(m.shape))
    f = capi.taccum(1.0, p["f"], -RATE, capi.orthogonalise(momentum).reshape(p["f"].shape))
    return dict(loss=loss, dx=dx, dg=dg, db=db, df=df, dfb=dfb, f=f)


def loss64(x, g, b, f, fb, c, w):
    N = x.shape[0]
    x = x.reshape(N, -1)
    mu = x.mean(dim=1, keepdim=True)
    y = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(dim=1, keepdim=True) + EPS) * g + b
    z = y @ f.reshape(f.shape[0], -1).t() + fb
    at = (c.long() - 1).clamp(min=0)
    terms = torch.logsumexp(z, dim=1) - z[torch.arange(N, device=z.device), at]
    return (torch.where(c > 0, terms * w, torch.zeros_like(terms))).sum() / N


def step64(x, p, c, w, m):
    leaves = [t.double().cpu().requires_grad_() for t in (x, p["g"], p["b"], p["f"], p["fb"])]
    loss = loss64(*leaves, c.cpu(), w.double().cpu())
    dx, dg, db, df, dfb = torch.autograd.grad(loss, leaves)
    q = MOMENTUM * m.double().cpu()[0] + df.reshape(m.shape[1:])
    q = q / torch.linalg.norm(q)
    tall = q.shape[0] > q.shape[1]
    q = q.t() if tall else q
    for _ in range(5):
        a = q @ q.t()
        q = 3.4445 * q + (-4.7750 * a + 2.0315 * (a @ a)) @ q
    q = q.t() if tall else q
    return dict(loss=loss.detach(), dx=dx, dg=dg, db=db, df=df, dfb=dfb, f=leaves[3].detach() - RATE * q.reshape(leaves[3].shape))


# A sum of n products carries n u of the sum of magnitudes, and magnitudes here exceed results by cancellation: an output of the
# normalisation is off by 80 u of its row's largest (64 + C/256 additions and the scale), a score by (C + 8) u sum |y f| + 80 u sum |y f|,
# which for rows of norm sqrt(C) and filters of norm 1 is at most (C + 88) u sqrt(C) |f|; P by twice that and every gradient, relative
# to the norm of the products it sums, by P's error, (K + N + C) u of the sums and the normalisation's 4 x 80 u once more.  In norms,
# with sqrt(C) <= 32 and |f| about 1, and a factor 4 for sums of magnitudes over sums: 4 (32 x 2 (C + 88) + K + N + 320) u.
def gradient_bound(N, C, K):
    return 4 * (2 * C ** 0.5 * (C + 88) + K + N + 320) * U


# The update multiplies the gradient's relative error by at most 3.4445 in each of five steps (the iteration's largest slope), over
# matrices whose norm is at most 1.21 sqrt(min(K, C)), and adds its own, which is smaller: 3.4445^5 = 485.
@pytest.mark.parametrize("N,C,K", [(32, 64, 100), (33, 257, 70), (7, 130, 1001)])
def test_step(capi, N, C, K):
    x, p, c, w, m = make(N, C, K)
    got, want = step(capi, x, p, c, w, m), step64(x, p, c, w, m)
    off = gradient_bound(N, C, K)
    for name in ("dx", "dg", "db", "df", "dfb"):
        g, e = got[name].double().cpu().reshape(-1), want[name].reshape(-1)
        away = float(torch.linalg.norm(g - e) / torch.linalg.norm(e))
        assert away <= off, (name, away, off)
    assert abs(float(got["loss"]) - float(want["loss"])) <= off * float(want["loss"]), (float(got["loss"]), float(want["loss"]))
    away = float(torch.linalg.norm(got["f"].double().cpu() - want["f"]))
    assert away <= 2 * 485 * off * RATE + U * float(torch.linalg.norm(want["f"])), away


def test_gradients_against_differences(capi):
    """The loss of the operators' own forward calls along a direction d in all leaves at once.  (L(h) - L(-h))/2h differs from
    <gradient, d> by the difference's own error, which is taken from the same difference in double precision, and by the two losses'
    errors over 2h: a score is off by 2 (C + 88) u |y| |f| with |y| <= 2 sqrt(C) and |f| <= 2 (as above; multipliers up to 1.5), a loss
    by twice that and weights of 1.5 at most: 3 x 2 x 112 x 4 x 4.9 u = 7.9e-4; over h = 0.05: 1.6e-2."""
    N, C, K, h = 64, 24, 11, 5e-2
    x, p, c, w, m = make(N, C, K, seed=3)
    got = step(capi, x, p, c, w, m)
    r = torch.Generator(device="cuda")
    r.manual_seed(7)
    names = [("dx", x), ("dg", p["g"]), ("db", p["b"]), ("df", p["f"]), ("dfb", p["fb"])]
    # the direction: the gradient itself plus noise, so that the derivative is far from zero
    ds = []
    for name, t in names:
        d = got[name].reshape(t.shape)
        d = d / torch.linalg.norm(d)
        n = torch.randn(t.shape, generator=r, device="cuda")
        d = d + 0.5 * n / torch.linalg.norm(n)
        ds.append(d / torch.linalg.norm(d))

    def at(s, double):
        return [t.double() + s * h * d.double() if double else t + s * h * d for (_, t), d in zip(names, ds)]

    def loss(s):
        xx, g, b, f, fb = at(s, False)
        y, _ = capi.lnorm_forward(xx, g, b, EPS)
        return float(capi.fcloss_forward(y, f, fb, c, instance_weights=w)[0])

    slope = (loss(1) - loss(-1)) / (2 * h)
    leaves = [t.cpu().requires_grad_() for t in at(0, True)]
    exact = [float(loss64(*[t.cpu() for t in at(s, True)], c.cpu(), w.double().cpu())) for s in (1, -1)]
    exact = (exact[0] - exact[1]) / (2 * h)
    grads = torch.autograd.grad(loss64(*leaves, c.cpu(), w.double().cpu()), leaves)
    away = abs(exact - sum(float((g * d.double().cpu()).sum()) for g, d in zip(grads, ds)))
    want = sum(float((got[name].reshape(t.shape).double() * d.double()).sum()) for (name, t), d in zip(names, ds))
    assert abs(slope - want) <= away + 1.6e-2, (slope, want, away)
    assert want > 0.2   # (ten times what is allowed for)


def test_captured_step(capi):
    """The whole step in one graph, replayed with other inputs in between, against eager calls: the same bits."""
    x, p, c, w, m = make(48, 96, 300, seed=1)
    step(capi, x, p, c, w, m)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(capi, x, p, c, w, m)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            held = step(capi, x, p, c, w, m)
    torch.cuda.synchronize()
    for seed in (2, 5, 9):
        x2, p2, c2, w2, m2 = make(48, 96, 300, seed=seed)
        for a, b in ((x, x2), (c, c2), (w, w2), (m, m2)):
            a.copy_(b)
        for k in p:
            p[k].copy_(p2[k])
        eager = step(capi, x2, p2, c2, w2, m2)
        graph.replay()
        torch.cuda.synchronize()
        for name in eager:
            assert torch.equal(eager[name], held[name]), (seed, name)


def test_two_streams_at_once(capi):
    """Two steps on two streams at once, many times over: the bits of each alone (no call shares its workspace with another)."""
    jobs = [make(64, 128, 500, seed=1), make(40, 200, 300, seed=2)]
    want = [step(capi, *j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(step(capi, *j))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for name in b:
                assert torch.equal(a[name], b[name]), name


def test_front_end(capi, vl):
    """vl_nnlnorm and vl_nnfcloss: the C calls' bits, labels and weights from the host as well, options by name in any case."""
    x, p, c, w, m = make(20, 70, 33, seed=4)
    y, mom = vl.vl_nnlnorm(x, p["g"], p["b"], "epsilon", EPS, nout=2)
    want, moments = capi.lnorm_forward(x, p["g"], p["b"], EPS)
    assert torch.equal(y, want) and torch.equal(mom.reshape(-1), moments.reshape(-1))
    assert torch.equal(vl.vl_nnlnorm(x, p["g"], p["b"], "Epsilon", EPS, "MOMENTS", mom), want)
    dy = torch.randn_like(y)
    got = vl.vl_nnlnorm(x, p["g"], p["b"], dy, "epsilon", EPS, nout=4)
    for a, b in zip(got, capi.lnorm_backward(x, p["g"], dy, EPS)):
        assert torch.equal(a, b)
    # the backward pass takes its moments itself, with its own number of threads to a row: each of the two means is off by at most
    # 65 u max|x| (64 + C/256 additions one behind the other), each deviation by 65 u of itself and, by its mean, 65 u max|x| x 65 u
    # max|x| / sigma, which is nothing; sigma <= 2 max|x|
    most = 2 * 65 * U * 2 * float(x.abs().max())
    assert float((got[3].reshape(-1) - moments.reshape(-1)).abs().max()) <= most

    loss, sums = vl.vl_nnfcloss(y, p["f"], p["fb"], c, "instanceweights", w, nout=2)
    a, b = capi.fcloss_forward(y, p["f"], p["fb"], c, instance_weights=w)
    assert tuple(loss.shape) == (1, 1) and torch.equal(loss.reshape(-1), a.reshape(-1)) and torch.equal(sums.reshape(-1), b)
    host = vl.vl_nnfcloss(y, p["f"], p["fb"], c.double().cpu(), "instanceWeights", w.cpu())
    assert torch.equal(host, loss)
    whole = vl.vl_nnfcloss(y, p["f"], p["fb"], c, "normalise", 0.0)
    assert torch.equal(whole.reshape(-1), capi.fcloss_forward(y, p["f"], p["fb"], c, normalise=False)[0].reshape(-1))
    empty = torch.empty((0,), device="cuda")
    assert torch.equal(vl.vl_nnfcloss(y, p["f"], p["fb"], c, empty), vl.vl_nnfcloss(y, p["f"], p["fb"], c))
    for extra, k in ((["logSums", sums], dict(log_sums=b)), ([], {})):
        got = vl.vl_nnfcloss(y, p["f"], p["fb"], c, 0.7, "instanceWeights", w, *extra)
        for a, e in zip(got, capi.fcloss_backward(y, p["f"], p["fb"], c, 0.7, instance_weights=w, **k)):
            assert torch.equal(a.reshape(-1), e.reshape(-1))
    dx, df, dfb = vl.vl_nnfcloss(y, p["f"], empty, c, 0.7)
    want = capi.fcloss_backward(y, p["f"], None, c, 0.7)
    assert torch.equal(dx, want[0].reshape(dx.shape)) and torch.equal(df, want[1].reshape(df.shape)) and dfb.numel() == 0


def test_front_end_refuses(vl):
    d = lambda *s: torch.zeros(tuple(reversed(s)), device="cuda")
    for args, message in [((d(1, 1, 8, 4), d(8), d(7)), "The BIASES size does not match the DATA depth."),
                          ((d(1, 1, 8, 4), d(8), d(8), "moments", d(1, 1, 8, 2)), "The MOMENTS size does not match the DATA pixels."),
                          ((d(1, 1, 8, 4), d(8), d(8), d(1, 1, 8, 3)), "DATA and DEROUTPUT do not have the same size.")]:
        with pytest.raises(vl.VlError) as e:
            vl.vl_nnlnorm(*args)
        assert e.value.message == message
    for dtype in (torch.float64, torch.bfloat16):
        with pytest.raises(vl.VlError):
            vl.vl_nnlnorm(d(1, 1, 8, 4).to(dtype), d(8).to(dtype), d(8).to(dtype))
    with pytest.raises(vl.VlError) as e:
        vl.vl_nnfcloss(d(1, 1, 8, 4), d(1, 1, 8, 10), d(10), d(3))   # (three labels for four images)
    assert e.value.message == "mcn_fcloss_forward: C does not have one label per image"
    with pytest.raises(vl.VlError):
        vl.vl_nnfcloss(d(1, 1, 8, 4).double(), d(1, 1, 8, 10).double(), d(10).double(), d(4))


def front_step(vl, x, p, c, w, m):
    """The same step through the front-end, up to the bank's derivative."""
    y, moments = vl.vl_nnlnorm(x, p["g"], p["b"], "epsilon", EPS, nout=2)
    loss, sums = vl.vl_nnfcloss(y, p["f"], p["fb"], c, "instanceWeights", w, nout=2)
    dy, df, dfb = vl.vl_nnfcloss(y, p["f"], p["fb"], c, 1.0, "instanceWeights", w, "logSums", sums)
    dx, dg, db = vl.vl_nnlnorm(x, p["g"], p["b"], dy, "epsilon", EPS, "moments", moments)
    return dict(loss=loss, dx=dx, dg=dg, db=db, df=df, dfb=dfb)


def test_front_end_on_two_streams_at_once(vl):
    """As test_two_streams_at_once, through the front-end."""
    jobs = [make(64, 128, 500, seed=1), make(40, 200, 300, seed=2)]
    want = [front_step(vl, *j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(front_step(vl, *j))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for name in b:
                assert torch.equal(a[name], b[name]), name


def test_front_end_captured(vl):
    """The front-end's calls in two graphs (each with memory of its own), replayed in turn with other inputs, against eager calls."""
    jobs = [make(48, 96, 300, seed=1), make(20, 150, 70, seed=2)]
    held = []
    for j in jobs:
        front_step(vl, *j)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = front_step(vl, *j)
        held.append((graph, out))
    for seed in (3, 4, 5):
        for j, shape, (graph, out) in zip(jobs, ((48, 96, 300), (20, 150, 70)), held):
            x, p, c, w, m = make(*shape, seed=seed)
            for a, b in ((j[0], x), (j[2], c), (j[3], w)):
                a.copy_(b)
            for k in p:
                j[1][k].copy_(p[k])
        for graph, _ in held:
            graph.replay()
        torch.cuda.synchronize()
        for j, (_, out) in zip(jobs, held):
            want = front_step(vl, *j)
            for name in want:
                assert torch.equal(want[name], out[name]), (seed, name)


@pytest.mark.parametrize("N,C,K", [(32, 64, 100), (33, 257, 70), (7, 130, 1001)])
def test_every_link_of_the_step(capi, N, C, K):
    """Each call of a step against its formulas in double precision on what the call before it gave, with the bounds that its own tests
    derive: nothing grows from link to link, so a result of 16 bits, or four Newton-Schulz steps instead of five, does not pass."""
    import test_gpu_fcloss
    import test_gpu_lnorm
    import test_gpu_ortho
    x, p, c, w, m = make(N, C, K)
    y, moments = capi.lnorm_forward(x, p["g"], p["b"], EPS)
    loss, sums = capi.fcloss_forward(y, p["f"], p["fb"], c, instance_weights=w)
    dy, df, dfb = capi.fcloss_backward(y, p["f"], p["fb"], c, 1.0, instance_weights=w, log_sums=sums)
    dx, dg, db = capi.lnorm_backward(x, p["g"], dy, EPS, moments=moments)
    momentum = capi.taccum(MOMENTUM, m, 1.0, df.reshape(m.shape))
    turned = capi.orthogonalise(momentum)
    f = capi.taccum(1.0, p["f"], -RATE, turned.reshape(p["f"].shape))
    for name, got in step(capi, x, p, c, w, m).items():   # (the step is these calls)
        assert torch.equal(got, dict(loss=loss, dx=dx, dg=dg, db=db, df=df, dfb=dfb, f=f)[name]), name
    norm = test_gpu_lnorm.Want(x, p["g"], p["b"], dy, EPS)
    test_gpu_lnorm.near(y, norm.back(norm.y), norm.back(norm.y_off), "y")
    for name, got in (("dx", dx), ("dg", dg), ("db", db)):
        want, off = getattr(norm, name), getattr(norm, name + "_off")
        test_gpu_lnorm.near(got, norm.back(want) if name == "dx" else want, norm.back(off) if name == "dx" else off, name)
    head = test_gpu_fcloss.Want(y, p["f"], p["fb"], c, w)
    for name, got in (("y", loss), ("dx", dy), ("df", df), ("db", dfb)):
        test_gpu_fcloss.near(got, getattr(head, name).reshape(-1, 1) if name == "y" else getattr(head, name), getattr(head, name + "_off"), name)
    # (the coefficients are held in single precision; a product, a sum: one rounding each)
    want = MOMENTUM * m.double() + df.double().reshape(m.shape)
    assert bool(((momentum.double() - want).abs() <= 2 * U * (MOMENTUM * m.double()).abs() + U * want.abs()).all())
    want, off = test_gpu_ortho.reference(momentum[0], 5)
    assert float(torch.linalg.norm(turned[0].double() - want)) <= off
    want = p["f"].double() - RATE * turned.double().reshape(p["f"].shape)
    assert bool(((f.double() - want).abs() <= 2 * U * (RATE * turned.double().reshape(p["f"].shape)).abs() + U * want.abs()).all())
    # what would not pass: four steps
    four, _ = test_gpu_ortho.reference(momentum[0], 4)
    assert float(torch.linalg.norm(turned[0].double() - four)) > 10 * off
