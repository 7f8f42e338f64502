"""Operators of a training step in which positions see one another, as cases that can be timed and compared.

Three families, each through the public entry points of `matconvnet_amd.capi` on device tensors:

  hnorm      the heads of queries and keys normalised and rotated by their positions along one or several axes: the outputs,
             or the outputs and all derivatives
  attention  softmax attention over packed sequences with grouped heads, causal or not: the output, or the output and all
             derivatives; also one query a sequence against many keys
  clip       the norm of all gradients of a network, and the gradients clipped to it

`listed()` holds the cases, `draw()` gives more of the same ranges.  With `own` false `run()` computes the operators in
elementary torch operations.
"""
import math
import random

import torch

own = False

EPSILON = 1e-6
BASE = 10000.0          # frequencies fall from 1 to 1/BASE

_TYPES = {"single": torch.float32, "bfloat16": torch.bfloat16}

# --------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # one new position of sixteen sequences, far along them: a matter of launches
        _hnorm("hnorm answers", D=128, heads=32, keyHeads=8, N=16, axes=1, type="bfloat16", what="forward", far=True),
        # the pixels of 32 images of 14 x 14, rows and columns
        _hnorm("hnorm images", D=64, heads=12, keyHeads=12, N=6272, axes=2, type="single", what="both"),
        # a training step's worth of video positions: time, rows, columns
        _hnorm("hnorm video bfloat16", D=128, heads=32, keyHeads=8, N=16384, axes=3, type="bfloat16", what="both"),
        # odd heads, a part of the channels rotated, neighbours paired, no norm
        _hnorm("hnorm odd", D=75, heads=7, keyHeads=7, N=5001, axes=1, type="single", what="both", pairs=24, normalise=False, neighbours=True),
        # every pixel of an image sees every other: many short sequences of one length
        _attention("attention images", D=64, heads=12, keyHeads=12, sequences=32, N=6272, type="bfloat16", what="step"),
        # packed sequences of different lengths, heads in groups of four
        _attention("attention packed", D=128, heads=32, keyHeads=8, sequences=13, N=8192, type="bfloat16", what="step", causal=True, ragged=5),
        # one long sequence: the matrix pipe's case
        _attention("attention long", D=128, heads=32, keyHeads=8, sequences=1, N=16384, type="bfloat16", what="step", causal=True),
        # odd everywhere, in single precision
        _attention("attention odd", D=75, heads=6, keyHeads=2, sequences=9, N=5001, type="single", what="step", causal=True, ragged=11),
        # one query of 64 sequences against the keys before it: the keys and values are read once and that is all
        _attention("attention answers", D=128, heads=32, keyHeads=8, sequences=64, N=64, M=262144, type="bfloat16", what="forward", causal=True,
                   ragged=3),
        # the banks of a residual unit: a matter of launches
        dict(name="clip banks", family="clip", network="spread", count=10, total=70000, low=0, most=1.0),
        # ResNet-50's gradients
        dict(name="clip ResNet-50", family="clip", network="ResNet-50", count=161, total=25557032, low=0, most=1.0),
        # a classifier's bank in bfloat16 beside single-precision gradients, many of them odd
        dict(name="clip classifier", family="clip", network="spread", count=300, total=600000007, low=2, most=1.0),
    ]


def _hnorm(name, D, heads, keyHeads, N, axes, type, what, pairs=None, normalise=True, neighbours=False, far=False):
    c = dict(family="hnorm", D=D, heads=heads, keyHeads=keyHeads, N=N, axes=axes, type=type, what=what, pairs=D // 2 if pairs is None else pairs,
             normalise=normalise, neighbours=neighbours, far=far)
    return dict(c, name=name) if name else c


def _attention(name, D, heads, keyHeads, sequences, N, type, what, M=None, causal=False, ragged=0):
    """M: keys of all sequences (None: as many as queries, which are the keys' own); ragged: 0 for sequences of one length."""
    c = dict(family="attention", D=D, heads=heads, keyHeads=keyHeads, sequences=sequences, N=N, M=N if M is None else M, type=type, what=what,
             causal=causal, ragged=ragged)
    return dict(c, name=name) if name else c


def _spread(rng, low, high):
    """A whole number of [low, high], its logarithm spread evenly."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    family = rng.choice(["hnorm", "attention", "attention", "clip"])
    if family == "hnorm":
        D, keyHeads, group = _spread(rng, 16, 256), _spread(rng, 1, 16), rng.choice([1, 1, 2, 4, 7])
        if rng.random() < 0.6:
            D = (D + 15) // 16 * 16
        N = _spread(rng, 1, max(1, min(16384, (1 << 26) // (D * keyHeads * (group + 1)))))
        return _hnorm(None, D=D, heads=keyHeads * group, keyHeads=keyHeads, N=N, axes=rng.randint(1, 3), type=rng.choice(["single", "bfloat16"]),
                      what=rng.choice(["forward", "both", "both"]), pairs=rng.choice([D // 2, D // 2, max(3, D // 4)]),
                      normalise=rng.random() < 0.7, neighbours=rng.random() < 0.4, far=rng.random() < 0.3)
    if family == "attention":
        D, keyHeads, group = rng.choice([rng.randint(16, 128), 64, 80, 96, 128]), _spread(rng, 1, 12), rng.choice([1, 1, 2, 4, 7])
        heads, type, sequences = keyHeads * group, rng.choice(["single", "bfloat16", "bfloat16"]), _spread(rng, 1, 64)
        if rng.random() < 0.3:      # one query a sequence
            M = _spread(rng, sequences, max(sequences, min(262144, (1 << 28) // (D * keyHeads))))
            return _attention(None, D=D, heads=heads, keyHeads=keyHeads, sequences=sequences, N=sequences, M=M, type=type, what="forward", causal=True,
                              ragged=rng.randint(1, 1 << 20))
        each = _spread(rng, 1, max(1, min(8192, 16384 // sequences, int(math.sqrt((1 << 33) / (D * heads * sequences))))))
        return _attention(None, D=D, heads=heads, keyHeads=keyHeads, sequences=sequences, N=each * sequences, type=type,
                          what=rng.choice(["forward", "step", "step"]), causal=rng.random() < 0.6, ragged=rng.choice([0, rng.randint(1, 1 << 20)]))
    total = _spread(rng, 1000, 200000000)
    return dict(family="clip", network="spread", count=_spread(rng, 1, min(500, total // 10)), total=total, low=rng.choice([0, 0, 2, 3]),
                most=rng.choice([1.0, 1.0, 1e6]))


def _lengths(case):
    """(queries, keys) of each sequence, lists; where sequences differ, one of them is empty if there are three or more"""
    n, N, M = case["sequences"], case["N"], case["M"]
    if not case["ragged"]:
        return [N // n] * n, [M // n] * n
    rng = random.Random(case["ragged"])
    one = N != M or N == n        # one query each, so one key at least
    share = [rng.uniform(0.2, 1.8) for _ in range(n)]
    if not one and n > 2:
        share[rng.randrange(n)] = 0.0
    keys = [int(M * s / sum(share)) for s in share]
    if one:
        keys = [max(1, k - 1) for k in keys]
    while sum(keys) > M:          # (a few sequences of one key each)
        keys[keys.index(max(keys))] -= 1
    keys[max(range(n), key=lambda i: share[i])] += M - sum(keys)
    return ([1] * n if one else keys), keys


def _sizes(case):
    """[(shape, type)] of the gradients"""
    if case["network"] == "ResNet-50":
        shapes = [(64, 3, 7, 7), (64,), (64,)]
        inner, last = 64, 64
        for units in (3, 4, 6, 3):
            for u in range(units):
                for shape in ((inner, last, 1, 1), (inner, inner, 3, 3), (4 * inner, inner, 1, 1)) + (((4 * inner, last, 1, 1),) if u == 0 else ()):
                    shapes += [shape, (shape[0],), (shape[0],)]
                last = 4 * inner
            inner *= 2
        return [(s, "single") for s in shapes + [(1000, 2048, 1, 1), (1000,)]]
    rng = random.Random(case["count"] * 1000003 + case["total"])
    share = [math.exp(rng.uniform(0, 7)) for _ in range(case["count"])]
    if case["count"] > 2:
        share[0] = 0.85 * sum(share) if case["low"] else share[0]    # a classifier's bank, most of a network
    sizes = [int(case["total"] * s / sum(share)) for s in share]
    # every low-th gradient, the bank first, in bfloat16
    return [((max(1, s),), "bfloat16" if case["low"] and i % case["low"] == 0 else "single") for i, s in enumerate(sizes)]


# ------------------------------------------------------------------------------------------ what a user has in hand


def prepare(case, seed):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=r, device="cuda")
    uniform = lambda low, high, *shape: low + (high - low) * torch.rand(shape, generator=r, device="cuda")
    state = {"case": case}
    if case["family"] == "hnorm":
        D, N, type = case["D"], case["N"], _TYPES[case["type"]]
        h, hk = case["heads"], case["keyHeads"]
        # a projection's output: queries, keys and values of a position side by side, channels of different scales
        fused = (normal(N, h + 2 * hk, D) * uniform(0.5, 2.0, 1, h + 2 * hk, D)).to(type)
        state["q"], state["k"] = fused[:, :h], fused[:, h:h + hk]
        state["gq"], state["gk"] = (uniform(0.5, 1.5, D), uniform(0.5, 1.5, D)) if case["normalise"] else (None, None)
        state["dyq"], state["dyk"] = normal(N, h, D).to(type), normal(N, hk, D).to(type)
        axes, at = case["axes"], torch.arange(N, device="cuda", dtype=torch.float64)
        side = 14
        state["positions"] = torch.stack([at + (1000003 if case["far"] else 0)] if axes == 1 else [at // side % side, at % side] if axes == 2
                                         else [at // (side * side), at // side % side, at % side], dim=1).contiguous()
        # each axis has its run of the pairs
        pair = torch.arange(case["pairs"], device="cuda", dtype=torch.float64)
        frequency = BASE ** (-pair / case["pairs"])
        axis = (pair * axes / case["pairs"]).long()
        state["frequencies"] = torch.stack([torch.where(axis == a, frequency, 0.0) for a in range(axes)]).contiguous()
    elif case["family"] == "attention":
        D, N, M, type = case["D"], case["N"], case["M"], _TYPES[case["type"]]
        # normalised queries and keys: scores of a deviation of about 1.5, a few channels of the values larger than the others
        state["q"] = (1.2 * normal(N, case["heads"], D)).to(type)
        state["k"] = (1.2 * normal(M, case["keyHeads"], D)).to(type)
        state["v"] = (normal(M, case["keyHeads"], D) * uniform(0.3, 2.0, 1, case["keyHeads"], D)).to(type)
        state["dy"] = normal(N, case["heads"], D).to(type)
        state["lengths"] = _lengths(case)
        starts = lambda lengths: torch.tensor([0] + lengths, device="cuda").cumsum(0).int()
        state["q_starts"] = starts(state["lengths"][0]) if case["ragged"] else None
        state["k_starts"] = starts(state["lengths"][1]) if case["ragged"] else None
    else:
        sizes = _sizes(case)
        state["ders"] = [(normal(*shape) * 10.0 ** float(torch.empty(1).uniform_(-5, -2, generator=torch.Generator().manual_seed(seed + i))))
                         .to(_TYPES[type]) for i, (shape, type) in enumerate(sizes)]
        # the clipped ones lie one behind the other, those of a type in one array
        state["arena"], state["out"] = _arena(state["ders"], lambda g: g.dtype)
        if own:
            from matconvnet_amd import capi
            state["list"] = capi.GradientList(state["ders"], state["out"])
    return state


def _arena(ders, type):
    """({name of a type: zeros for all gradients of it, each from a multiple of 64 values on}, the gradients' places there)"""
    at, places = {}, []
    for g in ders:
        name = "bfloat16" if g.dtype == torch.bfloat16 else "single"
        places.append((name, at.get(name, 0)))
        at[name] = at.get(name, 0) + (g.numel() + 63) // 64 * 64
    types = {name: type(next(g for g, (n, _) in zip(ders, places) if n == name)) for name in at}
    arena = {name: torch.zeros(n, dtype=types[name], device="cuda") for name, n in at.items()}
    return arena, [arena[name][start:start + g.numel()].view(g.shape) for g, (name, start) in zip(ders, places)]


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    family = state["case"]["family"]
    return _run_hnorm(state) if family == "hnorm" else _run_attention(state) if family == "attention" else _run_clip(state)


def _run_hnorm(s):
    c = s["case"]
    both = c["what"] == "both"
    if own:
        from matconvnet_amd import capi
        how = dict(epsilon=EPSILON, normalise=c["normalise"], neighbours=c["neighbours"])
        yq, yk = capi.hnorm_forward(s["q"], s["k"], s["gq"], s["gk"], s["positions"], s["frequencies"], **how)
        if not both:
            return {"yq": yq, "yk": yk}
        dq, dk, dgq, dgk = capi.hnorm_backward(s["q"], s["k"], s["gq"], s["gk"], s["positions"], s["frequencies"], s["dyq"], s["dyk"], **how)
        out = {"yq": yq, "yk": yk, "dq": dq, "dk": dk}
        return dict(out, dgq=dgq, dgk=dgk) if c["normalise"] else out
    # the angles in 64 bits: those of far positions keep few digits otherwise
    angle = s["positions"] @ s["frequencies"]
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    pairs = c["pairs"]

    def split(t):
        if c["neighbours"]:
            return t[..., 0:2 * pairs:2], t[..., 1:2 * pairs:2]
        return t[..., :pairs], t[..., pairs:2 * pairs]

    def turned(t, sin):
        lo, hi = split(t)
        a, b = lo * cos - hi * sin, hi * cos + lo * sin
        front = torch.stack([a, b], dim=-1).flatten(-2) if c["neighbours"] else torch.cat([a, b], dim=-1)
        return torch.cat([front, t[..., 2 * pairs:]], dim=-1)

    out = {}
    for which in "qk":
        x, g = s[which].float(), s["g" + which]
        if c["normalise"]:
            sigma = torch.sqrt(x.square().mean(dim=-1, keepdim=True) + EPSILON)
            xh = x / sigma
        out["y" + which] = turned(xh * g if c["normalise"] else x, sin).to(s[which].dtype)
        if both:
            du = turned(s["dy" + which].float(), -sin)
            if c["normalise"]:
                out["dg" + which] = (du * xh).sum(dim=(0, 1))
                a = du * g
                du = (a - xh * (a * xh).mean(dim=-1, keepdim=True)) / sigma
            out["d" + which] = du.to(s[which].dtype)
    return out


def _run_attention(s):
    c = s["case"]
    step = c["what"] == "step"
    if own:
        from matconvnet_amd import capi
        how = dict(sequences=c["sequences"], q_starts=s["q_starts"], k_starts=s["k_starts"], causal=c["causal"])
        y, log_sums = capi.attention_forward(s["q"], s["k"], s["v"], **how)
        if not step:
            return {"y": y, "log_sums": log_sums}
        dq, dk, dv = capi.attention_backward(s["q"], s["k"], s["v"], y, log_sums, s["dy"], **how)
        return {"y": y, "log_sums": log_sums, "dq": dq, "dk": dk, "dv": dv}
    group, D = c["heads"] // c["keyHeads"], c["D"]
    scale = 1.0 / math.sqrt(D)
    out = {"y": torch.empty_like(s["q"]), "log_sums": torch.empty(c["N"], c["heads"], device="cuda")}
    if step:
        out["dq"], out["dk"], out["dv"] = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
    n, m = s["lengths"]
    if not c["ragged"]:          # all sequences at once, as long as their scores are not too many
        batch = max(1, min(c["sequences"], (1 << 31) // (n[0] * m[0] * c["heads"])))
        parts = [(i, min(batch, c["sequences"] - i)) for i in range(0, c["sequences"], batch)]
    else:
        parts = [(i, 1) for i in range(c["sequences"])]
    for i, many in parts:
        nq, nk = n[i], m[i]
        if nq == 0:
            continue
        q0, k0 = sum(n[:i]), sum(m[:i])
        # key heads whose scores are held at a time
        some = max(1, min(c["keyHeads"], (1 << 31) // (many * group * nq * nk)))
        for h in range(0, c["keyHeads"], some):
            hs = min(some, c["keyHeads"] - h)
            # many x heads x (queries of the group, one head behind the other) x D
            queries = lambda t: (t[q0:q0 + many * nq, h * group:(h + hs) * group].float().view(many, nq, hs, group, D).permute(0, 2, 3, 1, 4)
                                 .reshape(many, hs, group * nq, D))
            keys = lambda t: t[k0:k0 + many * nk, h:h + hs].float().view(many, nk, hs, D).permute(0, 2, 1, 3).contiguous()
            rows = lambda t: t.view(many, hs, group, nq, -1).permute(0, 3, 1, 2, 4).reshape(many * nq, hs * group, -1)
            columns = lambda t: t.permute(0, 2, 1, 3).reshape(many * nk, hs, D)
            q, k, v = queries(s["q"]), keys(s["k"]), keys(s["v"])
            z = q @ k.transpose(2, 3)
            z *= scale
            if c["causal"]:      # the queries are the last positions of their sequence
                hidden = torch.arange(nk, device="cuda") > torch.arange(nq, device="cuda").view(nq, 1) + (nk - nq)
                z.view(many, hs, group, nq, nk).masked_fill_(hidden, -math.inf)
            most = z.max(dim=3, keepdim=True).values
            z -= most
            p = z.exp_()
            total = p.sum(dim=3, keepdim=True)
            p /= total
            y = p @ v
            out["y"][q0:q0 + many * nq, h * group:(h + hs) * group] = rows(y.to(s["q"].dtype))
            out["log_sums"][q0:q0 + many * nq, h * group:(h + hs) * group] = rows(most + torch.log(total)).squeeze(-1)
            if not step:
                continue
            dy = queries(s["dy"])
            out["dv"][k0:k0 + many * nk, h:h + hs] = columns(p.transpose(2, 3) @ dy).to(s["v"].dtype)
            dp = dy @ v.transpose(2, 3)
            dp -= (dy * y).sum(dim=3, keepdim=True)
            dp *= p
            dp *= scale
            out["dq"][q0:q0 + many * nq, h * group:(h + hs) * group] = rows(dp @ k).to(s["q"].dtype)
            out["dk"][k0:k0 + many * nk, h:h + hs] = columns(dp.transpose(2, 3) @ q).to(s["k"].dtype)
    return out


def _run_clip(s):
    if own:
        from matconvnet_amd import capi
        norm = capi.clip_gradients(s["list"], s["case"]["most"])
    else:
        # the squares' sum in 64 bits: hundreds of millions of terms
        total = torch.zeros((), dtype=torch.float64, device="cuda")
        for g in s["ders"]:
            total += g.float().square().sum(dtype=torch.float64)
        norm = total.sqrt()
        factor = torch.where(norm > s["case"]["most"], s["case"]["most"] / norm, 1.0).float()
        for g, y in zip(s["ders"], s["out"]):
            y.copy_(g.float() * factor)
        norm = norm.float().view(1)
    return dict(s["arena"], norm=norm)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["family"] == "hnorm":
        n, size = case["D"] * (case["heads"] + case["keyHeads"]) * case["N"], _TYPES[case["type"]].itemsize
        return {"bytes": n * size * (2 if case["what"] == "forward" else 4), "flops": n * (8 if case["what"] == "forward" else 24)}
    if case["family"] == "attention":
        n, m = _lengths(case)
        D, size, step = case["D"], _TYPES[case["type"]].itemsize, case["what"] == "step"
        pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(n, m)) * case["heads"]
        queries, keys = case["N"] * case["heads"] * D, case["M"] * case["keyHeads"] * D
        return {"bytes": size * (queries * (4 if step else 2) + keys * (4 if step else 2)), "flops": pairs * D * (14 if step else 4)}
    n = sum(math.prod(shape) * _TYPES[type].itemsize for shape, type in _sizes(case))
    return {"bytes": 2 * n, "flops": 3 * sum(math.prod(shape) for shape, _ in _sizes(case))}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["family"] == "hnorm":
            return _exact_hnorm(case, s)
        return _exact_attention(case, s) if case["family"] == "attention" else _exact_clip(case, s)


def _exact_hnorm(case, s):
    """Pairs of channels as complex numbers, turned by e^(i angle); the derivative by the Jacobian of a normalised row."""
    P, D, both = case["pairs"], case["D"], case["what"] == "both"
    lo = torch.arange(P, device="cuda") * (2 if case["neighbours"] else 1)
    hi = lo + (1 if case["neighbours"] else P)
    angle = (s["positions"].unsqueeze(2) * s["frequencies"].unsqueeze(0)).sum(dim=1).unsqueeze(1)
    turn = torch.polar(torch.ones_like(angle), angle)

    def rotated(t, turn):
        z = torch.complex(t[..., lo], t[..., hi]) * turn
        t = t.clone()
        t[..., lo], t[..., hi] = z.real, z.imag
        return t

    out = {}
    for w in "qk":
        x = s[w].double()
        g = s["g" + w].double() if case["normalise"] else None
        r = torch.rsqrt((x * x).sum(dim=-1, keepdim=True) / D + EPSILON) if case["normalise"] else None
        out["y" + w] = rotated(x * r * g if case["normalise"] else x, turn)
        if both:
            u = rotated(s["dy" + w].double(), turn.conj())
            if case["normalise"]:
                out["dg" + w] = torch.einsum("nhd,nhd,nh->d", u, x, r.squeeze(-1))
                a = u * g
                out["d" + w] = r * a - x * (r ** 3 / D) * (a * x).sum(dim=-1, keepdim=True)
            else:
                out["d" + w] = u
    return out


def _exact_attention(case, s):
    """Sequence by sequence and head by head; the softmax's derivative as P (dP - sum P dP)."""
    n, m = s["lengths"]
    heads, group, D, step = case["heads"], case["heads"] // case["keyHeads"], case["D"], case["what"] == "step"
    if 14 * sum(a * b for a, b in zip(n, m)) * heads * D > 4e14 or case["sequences"] * heads > 4096:
        return None
    scale = D ** -0.5
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")
    out = {"y": zeros(s["q"]), "log_sums": torch.zeros(case["N"], heads, dtype=torch.float64, device="cuda")}
    if step:
        out.update(dq=zeros(s["q"]), dk=zeros(s["k"]), dv=zeros(s["v"]))
    q0 = k0 = 0
    for nq, nk in zip(n, m):
        qs, ks = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        if nq == 0:
            continue
        seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda").tril(nk - nq) if case["causal"] else None
        for h in range(heads):
            q, k, v = s["q"][qs, h].double(), s["k"][ks, h // group].double(), s["v"][ks, h // group].double()
            z = torch.mm(q, k.t()).mul_(scale)
            if seen is not None:
                z = torch.where(seen, z, -math.inf)
            sums = torch.logsumexp(z, dim=1)
            p = torch.exp(z - sums.unsqueeze(1))
            out["y"][qs, h], out["log_sums"][qs, h] = torch.mm(p, v), sums
            if step:
                dy = s["dy"][qs, h].double()
                out["dv"][ks, h // group] += torch.mm(p.t(), dy)
                dp = torch.mm(dy, v.t())
                dz = p * (dp - (p * dp).sum(dim=1, keepdim=True)) * scale
                out["dq"][qs, h] = torch.mm(dz, k)
                out["dk"][ks, h // group] += torch.mm(dz.t(), q)
    return out


def _exact_clip(case, s):
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["ders"]))
    factor = min(1.0, case["most"] / norm)
    arena, places = _arena(s["ders"], lambda g: torch.float64)
    for g, y in zip(s["ders"], places):
        torch.mul(g.double(), factor, out=y)
    return dict(arena, norm=torch.tensor([norm], dtype=torch.float64, device="cuda"))
