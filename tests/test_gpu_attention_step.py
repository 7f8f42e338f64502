"""A training step of a small model in which positions see one another, out of the framework's operators as they would be used together:
layer normalisation, a projection (vl_nnconv's fully connected case over positions), heads normalised and rotated, attention over packed
sequences, an output projection and its sum with the input, a classifier with its loss; backward; gradients clipped and the solver's step.
Against the same in double precision by automatic differentiation on the CPU.

Every operator's own test bounds it element by element; what is looked at here is what they hand each other.  In single precision each is off by
some 2^-20 of its output's largest value and the convolutions by 2e-4 at most (their gate); five of them one behind the other stay
within 1e-3 of a gradient's largest value.  In bfloat16 the heads are rounded six times on the way (2^-8 each, halved by the mean over
channels and keys): 2^-5."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LENGTHS = [37, 0, 80, 1, 66]
N, C, HEADS, KEY_HEADS, D, CLASSES = sum(LENGTHS), 64, 6, 2, 40, 50
OUT = (HEADS + 2 * KEY_HEADS) * D


def parameters(seed=0):
    r = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=r)
    return {"g": 1 + 0.1 * normal(C), "b": 0.1 * normal(C), "wqkv": normal(OUT, C) / math.sqrt(C), "gq": 1 + 0.1 * normal(D), "gk": 1 + 0.1 * normal(D),
            "wo": normal(C, HEADS * D) / math.sqrt(HEADS * D), "f": normal(CLASSES, C) / math.sqrt(C), "bias": 0.1 * normal(CLASSES)}


def data(seed=1):
    r = torch.Generator().manual_seed(seed)
    x = torch.randn(N, C, generator=r)
    labels = torch.randint(0, CLASSES + 1, (N,), generator=r).float()
    at = torch.arange(N, dtype=torch.float64)
    return x, labels, torch.stack([at // 9, at % 9], dim=1)


def frequencies():
    f = torch.zeros(2, D // 2, dtype=torch.float64)
    for j in range(D // 2):
        f[j * 4 // D, j] = 10000.0 ** (-2 * j / D)
    return f


def by_differentiation(P, x, labels, positions):
    P = {k: v.double().requires_grad_() for k, v in P.items()}
    x = x.double().requires_grad_()
    xh = (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5)
    h = (xh * P["g"] + P["b"]) @ P["wqkv"].t()
    q, k, v = h.view(N, -1, D).split([HEADS, KEY_HEADS, KEY_HEADS], dim=1)
    angle = (positions @ frequencies()).unsqueeze(1)

    def heads(t, g):
        t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * g
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * torch.cos(angle) - b * torch.sin(angle), b * torch.cos(angle) + a * torch.sin(angle)], dim=-1)

    q, k = heads(q, P["gq"]), heads(k, P["gk"])
    rows, at = [], 0
    for n in LENGTHS:
        s = slice(at, at + n)
        at += n
        if n == 0:
            continue
        group = HEADS // KEY_HEADS
        K, V = k[s].repeat_interleave(group, dim=1), v[s].repeat_interleave(group, dim=1)
        z = torch.einsum("ihd,jhd->hij", q[s], K) / math.sqrt(D)
        z = z.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -math.inf)
        rows.append(torch.einsum("hij,jhd->ihd", torch.softmax(z, dim=-1), V))
    y = torch.cat(rows).reshape(N, -1) @ P["wo"].t() + x
    z = y @ P["f"].t() + P["bias"]
    on = labels > 0
    loss = (torch.logsumexp(z, 1) - z[torch.arange(N), (labels.long() - 1).clamp(min=0)])[on].sum() / N
    loss.backward()
    return float(loss.detach()), {k: v.grad for k, v in P.items()}, x.grad


def by_operators(capi, P, x, labels, positions, dtype):
    """The step with one contiguous arena of derivatives, as mcn_sgd_momentum takes it"""
    P = {k: v.cuda() for k, v in P.items()}
    counts = [v.numel() for v in P.values()]
    offsets, chunks, chunk_param = capi.sgd_arena_layout(counts)
    ders = torch.zeros(chunks * capi.SGD_CHUNK, device="cuda")
    places = {k: ders[o:o + n] for k, o, n in zip(P, offsets, counts)}
    rows = lambda t: t.reshape(t.shape[0], -1, 1, 1).contiguous()          # 1 x 1 x channels x positions
    x, labels, positions = x.cuda(), labels.cuda(), positions.cuda()
    f = frequencies().cuda()
    starts = torch.tensor(np.concatenate([[0], np.cumsum(LENGTHS)]), dtype=torch.int32, device="cuda")
    how = dict(q_starts=starts, k_starts=starts, causal=True)
    cast = lambda t: capi.convert(t, dtype) if t.dtype != dtype else t
    back = lambda t: capi.convert(t, torch.float32) if t.dtype != torch.float32 else t
    # forward
    xn, moments = capi.lnorm_forward(rows(x), P["g"], P["b"])
    g1 = capi.conv_geom((1, 1, C, N), (1, 1, C, OUT))
    h = cast(capi.conv_forward(xn, rows(P["wqkv"]), None, g1)).view(N, -1, D)
    parts = lambda t: (t[:, :HEADS], t[:, HEADS:HEADS + KEY_HEADS], t[:, HEADS + KEY_HEADS:])
    q, k, v = parts(h)
    yq, yk = capi.hnorm_forward(q, k, P["gq"], P["gk"], positions, f)
    y, sums = capi.attention_forward(yq, yk, v, **how)
    g2 = capi.conv_geom((1, 1, HEADS * D, N), (1, 1, HEADS * D, C))
    y1 = rows(back(y).view(N, -1))
    out = capi.add(capi.conv_forward(y1, rows(P["wo"]), None, g2), rows(x))
    loss, log_sums = capi.fcloss_forward(out, rows(P["f"]), P["bias"], labels)
    # backward
    dout, df, db = capi.fcloss_backward(out, rows(P["f"]), P["bias"], labels, log_sums=log_sums)
    dy1, dwo, _ = capi.conv_backward(y1, rows(P["wo"]), dout, g2, want=(True, True, False))
    dh = torch.empty_like(h)
    dq, dk, dv = parts(dh)
    dyq, dyk, _ = capi.attention_backward(yq, yk, v, y, sums, cast(dy1).view(N, HEADS, D), **dict(how, out=(torch.empty_like(yq), torch.empty_like(yk), dv)))
    _, _, dgq, dgk = capi.hnorm_backward(q, k, P["gq"], P["gk"], positions, f, dyq, dyk, out=(dq, dk))
    dxn, dwqkv, _ = capi.conv_backward(xn, rows(P["wqkv"]), rows(back(dh).view(N, -1)), g1, want=(True, True, False))
    dx, dg, dbeta = capi.lnorm_backward(rows(x), P["g"], dxn, moments=moments)
    dx = capi.add(dx, dout)
    for name, t in dict(g=dg, b=dbeta, wqkv=dwqkv, gq=dgq, gk=dgk, wo=dwo, f=df, bias=db).items():
        places[name].copy_(t.reshape(-1))
    # clipped, and the solver's step
    value = torch.zeros_like(ders)
    for (name, p), o in zip(P.items(), offsets):
        value[o:o + p.numel()] = p.reshape(-1)
    state, rates = torch.zeros_like(value), torch.ones(len(counts), 2, dtype=torch.float64, device="cuda")
    norm = capi.sgd_momentum_clipped(value, state, ders, torch.from_numpy(chunk_param).cuda(), rates, 0.1, 0.0, 0.9, 0.05)
    return loss, {k: t.clone() for k, t in places.items()}, dx.view(N, C), norm, {k: state[o:o + n].clone() for k, o, n in zip(P, offsets, counts)}


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 1e-3), (torch.bfloat16, 2.0 ** -5)])
def test_a_training_step(capi, dtype, bound):
    P, (x, labels, positions) = parameters(), data()
    loss, want, dx = by_differentiation(P, x, labels, positions)
    got_loss, got, got_dx, norm, state = by_operators(capi, P, x, labels, positions, dtype)
    assert abs(float(got_loss) - loss) <= bound * abs(loss)
    for name, t in want.items():
        off = (got[name].double().cpu().view(t.shape) - t).abs().max()
        assert float(off) <= bound * float(t.abs().max()), (name, float(off), float(t.abs().max()))
    assert float((got_dx.double().cpu() - dx).abs().max()) <= bound * float(dx.abs().max())
    # clipped to 0.05
    total = math.sqrt(sum(float(t.square().sum()) for t in want.values()))
    assert total > 0.05 and abs(float(norm) - total) <= bound * total
    moved = math.sqrt(sum(float(s.double().square().sum()) for s in state.values()))
    assert abs(moved - 0.05) <= 1e-6 * 0.05 * 16


def test_the_step_captured_into_a_graph(capi):
    """... and replayed among eager calls: the same bits"""
    P, (x, labels, positions) = parameters(), data()
    for dtype in (torch.float32, torch.bfloat16):
        at = {k: v.cuda() for k, v in P.items()}
        xs = x.cuda()
        torch.cuda.synchronize()
        starts = torch.tensor(np.concatenate([[0], np.cumsum(LENGTHS)]), dtype=torch.int32, device="cuda")
        f, pos = frequencies().cuda(), positions.cuda()
        h = (xs @ at["wqkv"].t()).to(dtype).view(N, -1, D)
        dy = torch.randn(N, HEADS, D, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(dtype)

        def step():
            q, k, v = h[:, :HEADS], h[:, HEADS:HEADS + KEY_HEADS], h[:, HEADS + KEY_HEADS:]
            yq, yk = capi.hnorm_forward(q, k, at["gq"], at["gk"], pos, f)
            y, sums = capi.attention_forward(yq, yk, v, q_starts=starts, k_starts=starts, causal=True)
            dyq, dyk, dv = capi.attention_backward(yq, yk, v, y, sums, dy, q_starts=starts, k_starts=starts, causal=True)
            dq, dk, dgq, dgk = capi.hnorm_backward(q, k, at["gq"], at["gk"], pos, f, dyq, dyk)
            outs = [torch.empty_like(t) for t in (dq, dk, dv, dgq, dgk)]
            norm = capi.clip_gradients(capi.GradientList([dq, dk, dv, dgq, dgk], outs), 0.1)
            return [y, norm] + outs

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        for i in range(3):
            h.copy_(torch.roll(h, 1, 0))
            eager = step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(captured, eager)), (dtype, i)
            for t in captured:
                t.zero_()
