"""vl_nnhnorm and vl_nnattention against the calls behind them, bit by bit: shapes, options, results that are not asked for, two streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(sequences=3, n=37, m=37, heads=6, keyHeads=2, D=40, seed=0):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=r, device="cuda")
    return normal(sequences, n, heads, D), normal(sequences, m, keyHeads, D), normal(sequences, m, keyHeads, D), normal(sequences, n, heads, D)


def flat(t):
    return t.flatten(0, 1)


def same(a, b):
    assert torch.equal(a.reshape(-1), b.reshape(-1))


def test_attention(capi, vl):
    for n, m, causal, scale in ((37, 37, False, None), (37, 37, True, 0.3), (1, 300, True, None), (5, 70, True, None)):
        q, k, v, dy = make(n=n, m=m)
        options = ["causal", float(causal)] + (["Scale", scale] if scale else [])
        how = dict(sequences=3, causal=causal, scale=scale)
        y, sums = vl.vl_nnattention(q, k, v, *options, nout=2)
        want, want_sums = capi.attention_forward(flat(q), flat(k), flat(v), **how)
        assert y.numel() == q.numel() and sums.numel() == want_sums.numel()
        same(y, want)
        same(sums, want_sums)
        same(vl.vl_nnattention(q, k, v, *options), want)
        ders = capi.attention_backward(flat(q), flat(k), flat(v), want, want_sums, flat(dy), **how)
        for extra in ([], ["OUTPUT", y.reshape(q.shape), "logsums", sums]):
            for a, b in zip(vl.vl_nnattention(q, k, v, dy, *options, *extra), ders):
                same(a, b)
        same(vl.vl_nnattention(q, k, v, dy, *options, nout=1), ders[0])


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("axes", [0, 1, 2])
def test_norms_and_rotations(capi, vl, axes, neighbours):
    q, k, _, dyq = make()
    dyk = torch.randn_like(k)
    N, D = q.shape[0] * q.shape[1], q.shape[3]
    gq, gk = torch.rand(D, device="cuda") + 0.5, torch.rand(D, device="cuda") + 0.5
    positions = frequencies = None
    options = ["epsilon", 1e-5, "neighbours", float(neighbours)]
    if axes:
        positions = torch.randint(0, 500, (N, axes), device="cuda").double()
        frequencies = capi.axis_frequencies([8] * axes, axes)
        options += ["positions", positions, "frequencies", frequencies]
    how = dict(epsilon=1e-5, neighbours=neighbours)
    empty = torch.empty((0,), device="cuda")
    want = capi.hnorm_forward(flat(q), flat(k), gq, gk, positions, frequencies, **how)
    for a, b in zip(vl.vl_nnhnorm(q, k, gq, gk, *options), want):
        same(a, b)
    same(vl.vl_nnhnorm(q, k, gq, gk, *options, nout=1), want[0])
    ders = capi.hnorm_backward(flat(q), flat(k), gq, gk, positions, frequencies, flat(dyq), flat(dyk), **how)
    for n in (4, 3, 2):
        for a, b in zip(vl.vl_nnhnorm(q, k, gq, gk, dyq, dyk, *options, nout=n), ders):
            same(a, b)
    # keys alone, without multipliers; rotations alone
    alone = vl.vl_nnhnorm(empty, k, empty, empty, *options)
    assert alone[0].numel() == 0
    same(alone[1], capi.hnorm_forward(None, flat(k), None, None, positions, frequencies, **how)[1])
    got = vl.vl_nnhnorm(empty, k, empty, empty, empty, dyk, *options)
    same(got[1], capi.hnorm_backward(None, flat(k), None, None, positions, frequencies, None, flat(dyk), **how)[1])
    assert got[0].numel() == 0 and got[2].numel() == 0 and got[3].numel() == 0
    for a, b in zip(vl.vl_nnhnorm(q, k, empty, empty, "normalise", 0.0, *options),
                    capi.hnorm_forward(flat(q), flat(k), None, None, positions, frequencies, normalise=False, **how)):
        same(a, b)


def step(vl, q, k, v, dy, g):
    yq, yk = vl.vl_nnhnorm(q, k, g, g)
    y, sums = vl.vl_nnattention(yq, yk, v, "causal", 1.0, nout=2)
    dq, dk, dv = vl.vl_nnattention(yq, yk, v, dy, "causal", 1.0, "output", y, "logSums", sums)
    return vl.vl_nnhnorm(q, k, g, g, dq, dk) + (dv,)


def test_two_streams_at_once(vl):
    jobs = [make(4, 100, 100, 8, 4, 64, seed=1), make(2, 257, 257, 4, 1, 96, seed=2)]
    jobs = [j + (torch.rand(j[0].shape[3], device="cuda") + 0.5,) for j in jobs]
    want = [step(vl, *j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(step(vl, *j))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


def test_refusals(vl):
    q, k, v, dy = make()
    g = torch.ones(40, device="cuda")
    for call, message in [(lambda: vl.vl_nnattention(q.double(), k.double(), v.double()), "vl_nnattention: only single precision is implemented on the HIP device"),
                          (lambda: vl.vl_nnattention(q[:, :, :5], k, v), "mcn_attention_forward: 5 heads over 2 key heads"),
                          (lambda: vl.vl_nnhnorm(q, k, g, g, "positions", torch.zeros(111, 2, dtype=torch.float64, device="cuda")),
                           "POSITIONS and FREQUENCIES are taken together."),
                          (lambda: vl.vl_nnhnorm(q, k, g, g, "positions", torch.zeros(111, 2, device="cuda"), "frequencies", torch.zeros(2, 8, device="cuda")),
                           "POSITIONS and FREQUENCIES are not of class DOUBLE on the device."),
                          (lambda: vl.vl_nnhnorm(q, k, g, g, "positions", torch.zeros(110, 2, dtype=torch.float64, device="cuda"), "frequencies",
                                                 torch.zeros(2, 8, dtype=torch.float64, device="cuda")),
                           "POSITIONS are not axes x positions or FREQUENCIES not pairs x axes.")]:
        with pytest.raises(vl.VlError) as e:
            call()
        assert e.value.message == message
