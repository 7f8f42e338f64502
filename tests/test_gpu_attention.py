"""Attention over packed sequences against its formulas in double precision, element by element.

Tolerances, with u = 2^-24 and h = 2^-8 where an operand or an output is bfloat16 (half a step of 2^-7), 0 in single precision.
  A score is a sum of D products in single precision: off by (D + 16) u (scale sum |q k| + |L|), the log sum L taken off in the same sum; an exponential
  adds its argument's rounding and its own, 2^-20 together at arguments of up to some tens.  So p is off by d = that of itself, and by h
  more where it is an operand; a sum over n terms by (n + 64) u of the sum of magnitudes; an output by h of itself.
  o:  (h + 2 d + (n + 64) u) sum p |v| + h |o|
  delta: sum |do| times what o is off, and (D + 16) u sum |do o|;  do.v likewise: together e;  ds = p (do.v - delta): (h + d) |ds| + p e
  dq, dk, dv: the sums of these with |k|, |q|, |do|, times scale, and h of the result."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def make(N, M, heads, keyHeads, D, dtype, seed=0, spread=1.2):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=r, device="cuda")
    return ((spread * normal(N, heads, D)).to(dtype), (spread * normal(M, keyHeads, D)).to(dtype), normal(M, keyHeads, D).to(dtype),
            normal(N, heads, D).to(dtype))


def starts(lengths, first=0):
    return torch.tensor(list(itertools.accumulate([first] + list(lengths))), dtype=torch.int32, device="cuda")


class Want:
    """The formulas in double over sequences (queries, keys) from the given first rows on, with bounds for each element"""

    def __init__(self, q, k, v, dy, lengths, causal, scale=None, q0=0, k0=0):
        h = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
        heads, group, D = q.shape[1], q.shape[1] // k.shape[1], q.shape[2]
        scale = scale or 1.0 / math.sqrt(D)
        double = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")
        names = dict(o=q, dq=q, dk=k, dv=v)
        for n, t in names.items():
            setattr(self, n, double(t))
            setattr(self, n + "_off", double(t))
        self.sums = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
        self.sums_off = self.sums.clone()
        for n, m in lengths:
            qs, ks = slice(q0, q0 + n), slice(k0, k0 + m)
            q0, k0 = q0 + n, k0 + m
            if n == 0:
                continue
            for head in range(heads):
                kh = head // group
                Q, K, V, dO = q[qs, head].double(), k[ks, kh].double(), v[ks, kh].double(), dy[qs, head].double()
                seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
                if causal:
                    seen = seen.tril(m - n)
                some = seen.any(dim=1) if m else torch.zeros(n, dtype=torch.bool, device="cuda")
                S = torch.where(seen, scale * (Q @ K.t()), -math.inf)
                L = torch.logsumexp(S, dim=1) if m else torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
                L0 = torch.where(some, L, 0.0)
                P = torch.where(seen, torch.exp(S - L0[:, None]), 0.0)
                size = scale * (Q.abs() @ K.abs().t()) + L0.abs()[:, None]
                d = torch.where(seen, (D + 16) * U * size + 2.0 ** -20, 0.0)
                worst = d.amax(dim=1, keepdim=True) if m else torch.zeros(n, 1, dtype=torch.float64, device="cuda")
                o = P @ V
                o_off = (P * (h + d + worst + (m + 64) * U)) @ V.abs() + h * o.abs()
                self.o[qs, head], self.o_off[qs, head] = o, o_off
                self.sums[qs, head], self.sums_off[qs, head] = L, (worst + (m + 64) * U).squeeze(1) + 4 * U * L0.abs()
                delta = (dO * o).sum(dim=1, keepdim=True)
                e = (dO.abs() * (o_off + (D + 16) * U * o.abs())).sum(dim=1, keepdim=True) + (D + 16) * U * (dO.abs() @ V.abs().t())
                dS = P * (dO @ V.t() - delta)
                dS_off = (h + d) * dS.abs() + P * e * (1 + h + d)
                n_u, m_u = (n * group + 64) * U, (m + 64) * U
                self.dq[qs, head] = scale * (dS @ K)
                self.dq_off[qs, head] = scale * ((dS_off + m_u * (dS.abs() + dS_off)) @ K.abs())
                self.dk[ks, kh] += scale * (dS.t() @ Q)
                self.dk_off[ks, kh] += scale * ((dS_off + n_u * (dS.abs() + dS_off)).t() @ Q.abs())
                self.dv[ks, kh] += P.t() @ dO
                self.dv_off[ks, kh] += (P * (h + d + n_u)).t() @ dO.abs()
        for n in ("dq", "dk", "dv"):
            setattr(self, n + "_off", getattr(self, n + "_off") + (h + 4 * U) * getattr(self, n).abs())


def near(got, want, off, what):
    got = got.double()
    assert bool(torch.isfinite(got).all()), what + " is not finite"
    bad = (got - want).abs() - (off + 1e-30)
    assert float(bad.max()) <= 0, (what, float(bad.max()), float((got - want).abs().max()), float(off.max()))


def check_all(capi, q, k, v, dy, lengths, causal, ragged=True, **more):
    n, m = [a for a, _ in lengths], [b for _, b in lengths]
    how = dict(q_starts=starts(n), k_starts=starts(m)) if ragged else dict(sequences=len(lengths))
    how.update(causal=causal, **more)
    w = Want(q, k, v, dy, lengths, causal, more.get("scale"))
    y, sums = capi.attention_forward(q, k, v, **how)
    assert y.dtype == q.dtype and y.shape == q.shape and sums.shape == q.shape[:2]
    empty = torch.isinf(w.sums)
    assert torch.equal(torch.isinf(sums) & (sums < 0), empty)
    near(torch.where(empty, 0.0, sums.double()), torch.where(empty, 0.0, w.sums), w.sums_off, "log sums")
    near(y, w.o, w.o_off, "o")
    dq, dk, dv = capi.attention_backward(q, k, v, y, sums, dy, **how)
    near(dv, w.dv, w.dv_off, "dv")
    near(dk, w.dk, w.dk_off, "dk")
    near(dq, w.dq, w.dq_off, "dq")
    return y, sums, dq, dk, dv


CASES = [  # D, heads, keyHeads, [(queries, keys)...], causal
    (64, 1, 1, [(1, 1)], False), (64, 1, 1, [(1, 1)], True), (16, 2, 1, [(5, 5)], True), (64, 2, 2, [(32, 32)], False), (128, 2, 2, [(33, 65)], False),
    (128, 1, 1, [(64, 64)], True), (128, 4, 2, [(65, 65)], True), (64, 3, 1, [(128, 128)], True), (128, 8, 1, [(129, 129)], True),
    (72, 2, 2, [(200, 200)], True), (80, 4, 1, [(31, 63)], True), (96, 5, 5, [(300, 300)], False), (40, 7, 1, [(97, 131)], True),
    (128, 6, 2, [(0, 0), (1, 1), (70, 70), (0, 5), (3, 0), (129, 129)], True), (64, 2, 1, [(7, 7), (0, 0), (64, 64), (65, 65), (2, 2)], False),
    (128, 2, 1, [(10, 3), (100, 40), (1, 0), (5, 5)], True),          # more queries than keys: rows that see nothing
    (64, 4, 4, [(40, 300), (1, 200), (129, 500)], True),
    (100, 3, 3, [(50, 50), (77, 77)], True), (75, 6, 2, [(33, 33), (150, 150)], True), (7, 2, 1, [(40, 41)], True), (1, 1, 1, [(9, 9)], False),
    (127, 2, 2, [(130, 130)], False), (65, 2, 1, [(64, 200)], True), (128, 33, 1, [(3, 70)], True), (128, 66, 2, [(1, 300), (2, 129)], True),
    (24, 1, 1, [(513, 513)], True), (128, 2, 2, [(700, 700)], True),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_both_directions(capi, case, dtype):
    D, heads, keyHeads, lengths, causal = CASES[case]
    q, k, v, dy = make(sum(a for a, _ in lengths), sum(b for _, b in lengths), heads, keyHeads, D, dtype, case)
    check_all(capi, q, k, v, dy, lengths, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,m,sequences,causal", [(14 * 14, 14 * 14, 3, False), (49, 49, 5, True), (1, 100, 4, True), (3, 1, 2, False), (130, 70, 1, True)])
def test_sequences_of_one_length(capi, n, m, sequences, causal, dtype):
    q, k, v, dy = make(n * sequences, m * sequences, 4, 2, 64, dtype, n)
    check_all(capi, q, k, v, dy, [(n, m)] * sequences, causal, ragged=False)
    check_all(capi, q, k, v, dy, [(n, m)] * sequences, causal, ragged=False, scale=0.4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,keyHeads,D,keys", [(8, 2, 128, [5000]), (4, 4, 64, [1, 0, 2111, 700, 64]), (32, 8, 128, [900, 3333, 1, 129]), (7, 1, 75, [4001, 17]),
                                                   (40, 1, 128, [6000])])
def test_one_query_and_many_keys(capi, heads, keyHeads, D, keys, dtype):
    """Keys cut into slices that are put together: as near as whole ones; sequences shorter than a slice, or empty, among them"""
    lengths = [(1, m) for m in keys]
    q, k, v, dy = make(len(keys), sum(keys), heads, keyHeads, D, dtype, len(keys))
    check_all(capi, q, k, v, dy, lengths, True)


def test_many_sequences(capi):
    """More than 64, and more than 64 x 64, sequences: the search for a tile's sequence takes one, two and three steps"""
    for count in (64, 65, 200, 4097, 4500):
        lengths = [(i % 3, i % 3) for i in range(count)]
        n = sum(a for a, _ in lengths)
        q, k, v, dy = make(n, n, 1, 1, 16, torch.float32, count)
        s = starts([a for a, _ in lengths])
        y, sums = capi.attention_forward(q, k, v, q_starts=s, k_starts=s)
        grads = capi.attention_backward(q, k, v, y, sums, dy, q_starts=s, k_starts=s)
        # sequences of one and of two positions, all at once
        one = [sum(a for a, _ in lengths[:i]) for i in range(1, count, 3)]
        two = [sum(a for a, _ in lengths[:i]) for i in range(2, count, 3)]
        # (one key: o = (p v) (1/p) with p within 2^-20 of 1; p v, 1/p and their product are rounded once each: 3 u of |v|)
        near(y[one], v[one].double(), 3 * U * v[one].abs().double(), "o of one key")
        at = torch.tensor(two, device="cuda")
        a, b = torch.stack([at, at + 1]), torch.stack([at + 1, at])
        s0 = (q[a].double() * k[a].double()).sum(-1) / 4
        s1 = (q[a].double() * k[b].double()).sum(-1) / 4
        p = torch.sigmoid(s0 - s1).unsqueeze(-1)
        near(y[a], p * v[a].double() + (1 - p) * v[b].double(), 1e-5 * (v[a].abs() + v[b].abs()).double(), "o")
        near(sums[a], torch.logaddexp(s0, s1), 1e-5 * (1 + s0.abs() + s1.abs()), "log sums")
        assert all(bool(torch.isfinite(g).all()) for g in grads)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(capi, dtype):
    """Parts of a projection's output, heads ahead of positions, an odd first address, keys shared by stride 0, outputs of any strides: the same bits
    as contiguous tensors' where both are read alike, within the bounds otherwise"""
    lengths, causal = [(70, 70), (130, 130)], True
    s = starts([70, 130])
    n, heads, keyHeads, D = 200, 6, 2, 64
    q, k, v, dy = make(n, n, heads, keyHeads, D, dtype, 5)
    how = dict(q_starts=s, k_starts=s, causal=causal)
    y, sums = capi.attention_forward(q, k, v, **how)
    want = (y, sums) + capi.attention_backward(q, k, v, y, sums, dy, **how)

    def run(q, k, v, dy, out=None):
        y, sums = capi.attention_forward(q, k, v, out=None if out is None else out[0], **how)
        return (y, sums) + tuple(capi.attention_backward(q, k, v, y, sums, dy, out=None if out is None else out[1:], **how))

    fused = torch.cat([q, k, v], dim=1)
    part = lambda t: (t[:, :heads], t[:, heads:heads + keyHeads], t[:, heads + keyHeads:])
    assert all(torch.equal(a, b) for a, b in zip(run(*part(fused), dy), want))
    # ... and derivatives written into one
    dfused = torch.full_like(fused, 7.0)
    y2 = torch.full((heads, n, D), 7.0, dtype=dtype, device="cuda").transpose(0, 1)
    got = run(*part(fused), dy, out=(y2,) + part(dfused))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, dy)]
    assert all(torch.equal(a, b) for a, b in zip(run(*turned), want))

    def shifted(t):   # by one value
        room = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:] = t.reshape(-1)
        return room[1:].view(t.shape)

    def wide(t):      # rows of one value more than the heads take
        room = torch.full((t.shape[0], t.shape[1] * t.shape[2] + 1), 9.0, dtype=t.dtype, device="cuda")
        room[:, :-1] = t.reshape(t.shape[0], -1)
        return room.as_strided(t.shape, (room.shape[1], t.shape[2], 1))

    for how_laid in (shifted, wide):
        assert all(torch.equal(a, b) for a, b in zip(run(*[how_laid(t) for t in (q, k, v, dy)]), want))
        outs = tuple(how_laid(torch.zeros_like(t)) for t in (q, q, k, v))
        got = run(q, k, v, dy, out=outs)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one key head for both groups, by a stride of 0
    k1, v1 = k[:, :1].expand(n, keyHeads, D), v[:, :1].expand(n, keyHeads, D)
    a, b = run(q, k1, v1, dy), run(q, k1.contiguous(), v1.contiguous(), dy)
    assert all(torch.equal(x, z) for x, z in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_no_sequence_are_left_alone(capi, dtype):
    q, k, v, dy = make(150, 160, 4, 2, 80, dtype, 3)
    lengths = [(50, 60), (20, 20), (40, 40)]
    qs, ks = starts([n for n, _ in lengths], 13), starts([m for _, m in lengths], 9)
    w = Want(q, k, v, dy, lengths, True, q0=13, k0=9)
    inside = torch.zeros(150, dtype=torch.bool, device="cuda")
    inside[13:123] = True
    kinside = torch.zeros(160, dtype=torch.bool, device="cuda")
    kinside[9:129] = True
    how = dict(q_starts=qs, k_starts=ks, causal=True)
    # whatever other rows hold
    for t, keep in ((q, inside), (k, kinside), (v, kinside), (dy, inside)):
        t[~keep] = math.nan
    out = torch.full_like(q, 5.0)
    y, sums = capi.attention_forward(q, k, v, out=out, **how)
    assert y is out and bool((y[~inside] == 5.0).all())
    near(y[inside], w.o[inside], w.o_off[inside], "o")
    outs = [torch.full_like(t, 5.0) for t in (q, k, v)]
    got = capi.attention_backward(q, k, v, y, sums, dy, out=outs, **how)
    for g, name, keep in zip(got, ("dq", "dk", "dv"), (inside, kinside, kinside)):
        assert bool((g[~keep] == 5.0).all())
        near(g[keep], getattr(w, name)[keep], getattr(w, name + "_off")[keep], name)
    # fresh ones hold zeros there
    y, sums = capi.attention_forward(q, k, v, **how)
    got = capi.attention_backward(q, k, v, y, sums, dy, **how)
    assert bool((y[~inside] == 0).all()) and all(bool((g[~keep] == 0).all()) for g, keep in zip(got, (inside, kinside, kinside)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_has_no_part(capi, dtype, bad):
    """A key, a value, a query and a derivative that are not finite reach the rows that see them and no others"""
    n, at = 100, 77
    q, k, v, dy = make(n, n, 4, 2, 64, dtype, 8)
    how = dict(causal=True)
    y, sums = capi.attention_forward(q, k, v, **how)
    dq, dk, dv = capi.attention_backward(q, k, v, y, sums, dy, **how)
    w = Want(q, k, v, dy, [(n, n)], True)
    before, behind = slice(0, at), slice(at + 1, n)
    k2, v2 = k.clone(), v.clone()
    k2[at], v2[at, :, 3] = bad, bad
    y2, sums2 = capi.attention_forward(q, k2, v2, **how)
    near(y2[before], w.o[before], w.o_off[before], "o")
    assert torch.equal(sums2[before], sums[before])
    assert not bool(torch.isfinite(y2[at:, :, 3]).any())
    dq2, _, _ = capi.attention_backward(q, k2, v2, y2, sums2, dy, **how)
    near(dq2[before], w.dq[before], w.dq_off[before], "dq")
    # a query and its derivative: keys behind it are not seen by it
    q3, dy3 = q.clone(), dy.clone()
    q3[at], dy3[at, :, 5] = bad, bad
    y3, sums3 = capi.attention_forward(q3, k, v, **how)
    assert torch.equal(y3[before], y[before]) and torch.equal(y3[behind], y[behind])
    dq3, dk3, dv3 = capi.attention_backward(q3, k, v, y3, sums3, dy3, **how)
    near(dk3[behind], w.dk[behind], w.dk_off[behind], "dk")
    near(dv3[behind], w.dv[behind], w.dv_off[behind], "dv")
    near(dq3[behind], w.dq[behind], w.dq_off[behind], "dq")
    assert not bool(torch.isfinite(dv3[:at + 1, :, 5]).any())


def test_large_scores(capi):
    """Scores of hundreds of times the usual, and one key far above the others: nothing overflows, the winner takes all"""
    for dtype in TYPES:
        q, k, v, dy = make(90, 90, 2, 2, 128, dtype, 1, spread=30.0)
        check_all(capi, q, k, v, dy, [(90, 90)], True)
        q = torch.ones(40, 1, 64, dtype=dtype, device="cuda")
        k = -1e4 * torch.ones(200, 1, 64, dtype=dtype, device="cuda")
        k[150] = 1e4
        v = torch.randn(200, 1, 64, device="cuda").to(dtype)
        y, sums = capi.attention_forward(q, k, v)
        # (one key is all there is: o = (p v) (1/p), three roundings; in bfloat16 p is rounded in the product and not in the sum, and so is o)
        h = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
        want = v[150].double().expand(40, 1, 64)
        near(y, want, (2 * h + h * h + 4 * U) * want.abs(), "o of the winner")


def test_derivatives_against_differences(capi):
    """The derivatives in single precision against differences of the forward call's outputs, along random directions"""
    lengths = [(20, 33), (45, 45)]
    q, k, v, dy = make(65, 78, 4, 2, 32, torch.float32, 2, spread=0.7)
    how = dict(q_starts=starts([20, 45]), k_starts=starts([33, 45]), causal=True)
    y, sums = capi.attention_forward(q, k, v, **how)
    grads = capi.attention_backward(q, k, v, y, sums, dy, **how)
    step = 2.0 ** -6
    for which in range(3):
        direction = torch.randn(q.shape if which == 0 else k.shape, generator=torch.Generator(device="cuda").manual_seed(which), device="cuda")
        values = []
        for sign in (1, -1):
            moved = [t + sign * step * direction if i == which else t for i, t in enumerate((q, k, v))]
            values.append((capi.attention_forward(*moved, **how)[0].double() * dy.double()).sum())
        difference = float(values[0] - values[1]) / (2 * step)
        want = float((grads[which].double() * direction.double()).sum())
        # the third derivative along a direction of this size times step^2 / 6, and single precision's outputs over the step
        size = float((grads[which].double() * direction.double()).abs().sum())
        assert abs(difference - want) <= 5e-3 * size, (which, difference, want, size)


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_repeats_and_own_workspaces(capi, dtype):
    q, k, v, dy = make(300, 300, 4, 2, 128, dtype, 4)
    how = dict(sequences=2, causal=True)
    y, sums = capi.attention_forward(q, k, v, **how)
    full = capi.attention_backward(q, k, v, y, sums, dy, **how)
    ws = capi.Workspace()
    for want in itertools.product([True, False], repeat=3):
        got = capi.attention_backward(q, k, v, y, sums, dy, want=want, ws=ws, **how)
        for g, f, wanted in zip(got, full, want):
            assert (g is None) != wanted and (g is None or torch.equal(g, f))
    again = capi.attention_forward(q, k, v, ws=ws, **how)
    assert torch.equal(again[0], y) and torch.equal(again[1], sums)


def test_streams_and_graphs(capi):
    """Calls on two streams at once and a captured step, replayed among eager calls: the same bits"""
    shapes = [(400, 400, 4, 2, 128, torch.bfloat16), (8, 4000, 8, 2, 128, torch.bfloat16), (300, 300, 2, 2, 75, torch.float32)]
    for N, M, heads, keyHeads, D, dtype in shapes:
        sequences = 8 if N == 8 else 2
        q, k, v, dy = make(N, M, heads, keyHeads, D, dtype, 6)
        how = dict(sequences=sequences, causal=True)

        def step():
            y, sums = capi.attention_forward(q, k, v, **how)
            return (y, sums) + tuple(capi.attention_backward(q, k, v, y, sums, dy, **how))

        want = step()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = []
        for _ in range(3):
            for s in streams:
                s.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(s):
                    got.append(step())
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
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


def test_refusals(capi):
    q, k, v, dy = make(8, 8, 4, 2, 16, torch.float32)
    s = starts([3, 5])
    for bad in [lambda: capi.attention_forward(q, k, v[:4]), lambda: capi.attention_forward(q, k[:, :, :8], v[:, :, :8]),
                lambda: capi.attention_forward(q, k, v, q_starts=s), lambda: capi.attention_forward(q, k, v, sequences=3),
                lambda: capi.attention_forward(q, k, v, q_starts=s, k_starts=s[:2]), lambda: capi.attention_forward(q, k, v, scale=-1.0),
                lambda: capi.attention_forward(q, k, v, q_starts=s, k_starts=s, sequences=5), lambda: capi.attention_forward(q.cpu(), k, v),
                lambda: capi.attention_forward(q[:, :, ::2], k[:, :, ::2], v[:, :, ::2]), lambda: capi.attention_forward(q[0], k, v),
                lambda: capi.attention_forward(q, k, v, out=q[:4])]:
        with pytest.raises(ValueError):
            bad()
    for bad in [lambda: capi.attention_forward(q, k.bfloat16(), v), lambda: capi.attention_forward(q.half(), k.half(), v.half()),
                lambda: capi.attention_forward(q, k, v, q_starts=s.long(), k_starts=s.long())]:
        with pytest.raises(TypeError):
            bad()
    three = torch.randn(8, 3, 16, device="cuda")
    with pytest.raises(capi.McnError) as e:
        capi.attention_forward(three, k, v)
    assert e.value.code == capi.ILLEGAL_ARGUMENT
    wide = torch.randn(8, 2, 129, device="cuda")
    with pytest.raises(capi.McnError) as e:
        capi.attention_forward(wide, wide, wide)
    assert e.value.code == capi.UNSUPPORTED
    same = torch.zeros(1, 4, 16, device="cuda").expand(8, 4, 16)
    with pytest.raises(capi.McnError):
        capi.attention_forward(q, k, v, out=same)


def test_nothing_to_do(capi):
    for N, M in ((0, 0), (0, 5), (5, 0)):
        q, k, v, dy = make(N, M, 2, 1, 16, torch.bfloat16)
        y, sums = capi.attention_forward(q, k, v)
        assert bool((y == 0).all()) and bool((sums == -math.inf).all())
        for g in capi.attention_backward(q, k, v, y, sums, dy):
            assert bool((g == 0).all())


def test_a_cache_behind_the_32nd_bit(capi):
    """Keys and values whose last rows lie more than 2^32 bytes behind their first"""
    M, D = 1 << 20, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough memory")
    k = torch.zeros(M, 20, D, dtype=torch.bfloat16, device="cuda")     # 5.4 GB
    k[:, 1] = torch.randn(M, D, device="cuda").bfloat16()
    v = torch.zeros_like(k)
    v[:, 1] = torch.randn(M, D, device="cuda").bfloat16()
    q = torch.randn(2, 20, D, device="cuda").bfloat16()
    qs, ks = starts([1, 1]), starts([M - 700, 700])
    y, sums = capi.attention_forward(q, k, v, q_starts=qs, k_starts=ks)
    w = Want(q[1:, 1:2], k[M - 700:, 1:2].contiguous(), v[M - 700:, 1:2].contiguous(), q[1:, 1:2], [(1, 700)], False)
    near(y[1:, 1:2], w.o, w.o_off, "o")
    w = Want(q[:1, 1:2], k[:M - 700, 1:2].contiguous(), v[:M - 700, 1:2].contiguous(), q[:1, 1:2], [(1, M - 700)], False)
    near(y[:1, 1:2], w.o, w.o_off, "o")
    near(sums[:1, 1:2], w.sums, w.sums_off, "log sums")


@pytest.mark.parametrize("dtype", TYPES)
def test_what_all_see_is_not_mended(capi, dtype):
    """A value that is not finite in the first key reaches every row, beside one in the last key that reaches the last row alone"""
    n = 200
    q, k, v, dy = make(n, n, 2, 1, 128, dtype, 9)
    v[0, :, 7], v[n - 1, :, 9] = math.nan, math.inf
    y, sums = capi.attention_forward(q, k, v, causal=True)
    assert bool(torch.isnan(y[:, :, 7]).all()) and bool(torch.isfinite(sums).all())
    keep = torch.ones(128, dtype=torch.bool, device="cuda")
    keep[7] = keep[9] = False
    v2 = v.clone()
    v2[0, :, 7], v2[n - 1, :, 9] = 0.0, 0.0
    w = Want(q, k, v2, dy, [(n, n)], True)
    near(y[:, :, keep], w.o[:, :, keep], w.o_off[:, :, keep], "o")
    assert not bool(torch.isfinite(y[n - 1, :, 9]).any())
