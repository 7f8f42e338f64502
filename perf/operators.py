"""Operators at the end of a training step of a classifier with many classes, as cases that can be timed and compared.

Three families, each through the public entry points of `matconvnet_amd.capi` on device tensors (a MATLAB array
H x W x C x N is a contiguous tensor of shape (N, C, W, H)):

  lnorm   layer normalisation of every pixel's channels: the output, or the output and all derivatives
  fcloss  softmax cross entropy behind a fully connected layer, without a tensor of scores: the value, or the value and
          all derivatives
  ortho   filter banks (one matrix of `rows` filters each) orthogonalised by Newton-Schulz products

`listed()` holds the cases, `draw()` gives more of the same ranges.  With `own` false `run()` computes the operators in
elementary torch operations.
"""
import math

import torch

own = False

EPSILON = 1e-5
STEPS = 5                                # Newton-Schulz products ...
A, B, C = 3.4445, -4.7750, 2.0315        # ... X <- A X + B (X X') X + C (X X')^2 X

_TYPES = {"single": torch.float32, "bfloat16": torch.bfloat16}

# --------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # the pooled features of a ResNet-50 batch: a matter of launches
        _lnorm("lnorm features", C=2048, N=32, type="single", what="forward"),
        # a sequence model's activations, a training step's worth of positions
        _lnorm("lnorm positions bfloat16", C=4096, N=8192, type="bfloat16", what="both"),
        # odd channels and an odd number of positions in single precision: rows that start anywhere
        _lnorm("lnorm odd", C=1023, N=5001, type="single", what="both"),
        # the pixels of the widest tensor of a residual unit: channels a plane apart
        _lnorm("lnorm pixels", H=56, W=56, C=256, N=32, type="single", what="both"),
        # the head of ResNet-50 at its batch: 1000 classes, small
        _fcloss("fcloss 1000 classes", D=2048, K=1000, N=32, type="single", what="step"),
        # a training step over a vocabulary: the matrix pipe's case, in single precision and in bfloat16
        _fcloss("fcloss vocabulary", D=1024, K=32000, N=2048, type="single", what="step"),
        _fcloss("fcloss vocabulary bfloat16", D=4096, K=128000, N=8192, type="bfloat16", what="step"),
        # odd everywhere, a bias, instances without a label and with weights
        _fcloss("fcloss odd", D=1001, K=21841, N=1021, type="bfloat16", what="step", bias=True, skipped=True),
        # a small batch of answers scored: the filters are read once and that is all
        _fcloss("fcloss scored", D=4096, K=128000, N=64, type="bfloat16", what="forward"),
        # the 3x3 banks of a residual network's first section: a matter of launches
        dict(name="ortho small banks", family="ortho", rows=64, cols=576, count=3),
        # a classifier's weights, odd and tall
        dict(name="ortho tall", family="ortho", rows=2501, cols=777, count=1),
        # the largest square weights
        dict(name="ortho square", family="ortho", rows=4096, cols=4096, count=1),
    ]


def _lnorm(name, C, N, type, what, H=1, W=1):
    c = dict(family="lnorm", H=H, W=W, C=C, N=N, type=type, what=what)
    return dict(c, name=name) if name else c


def _fcloss(name, D, K, N, type, what, bias=False, skipped=False):
    c = dict(family="fcloss", D=D, K=K, N=N, type=type, what=what, bias=bias, skipped=skipped)
    return dict(c, name=name) if name else c


def _spread(rng, low, high):
    """A whole number of [low, high], its logarithm spread evenly."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    family = rng.choice(["lnorm", "fcloss", "ortho"])
    if family == "lnorm":
        H, W = (1, 1) if rng.random() < 0.7 else (_spread(rng, 2, 56), _spread(rng, 2, 56))
        C = _spread(rng, 8, 8192 if H * W == 1 else 1024)
        N = _spread(rng, 1, max(1, min(8192, (1 << 25) // (H * W * C))))
        return _lnorm(None, C=C, N=N, H=H, W=W, type=rng.choice(["single", "bfloat16"]), what=rng.choice(["forward", "both", "both"]))
    if family == "fcloss":
        type, what = rng.choice(["single", "bfloat16"]), rng.choice(["forward", "step", "step"])
        D, K = _spread(rng, 16, 4096), _spread(rng, 10, 128000)
        N = _spread(rng, 1, max(1, min(8192, (1 << 39) // (D * K))))
        return _fcloss(None, D=D, K=K, N=N, type=type, what=what, bias=rng.random() < 0.5, skipped=rng.random() < 0.3)
    rows, cols = _spread(rng, 8, 4096), _spread(rng, 8, 4096)
    count = _spread(rng, 1, max(1, min(16, (1 << 33) // (rows * cols * min(rows, cols)))))
    return dict(family="ortho", rows=rows, cols=cols, count=count)


# ------------------------------------------------------------------------------------------ what a user has in hand


def prepare(case, seed):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=r, device="cuda")
    uniform = lambda low, high, *shape: low + (high - low) * torch.rand(shape, generator=r, device="cuda")
    state = {"case": case}
    if case["family"] == "lnorm":
        shape, type = (case["N"], case["C"], case["W"], case["H"]), _TYPES[case["type"]]
        # channels of different scales and offsets, as activations have them
        scale, offset = uniform(0.5, 2.0, 1, case["C"], 1, 1), normal(1, case["C"], 1, 1)
        state["x"] = (normal(*shape) * scale + offset).to(type)
        state["dzdy"] = normal(*shape).to(type)
        state["g"], state["b"] = uniform(0.5, 1.5, case["C"]), 0.1 * normal(case["C"])
    elif case["family"] == "fcloss":
        D, K, N, type = case["D"], case["K"], case["N"], _TYPES[case["type"]]
        # normalised features, filters that give scores of a deviation of 2
        state["x"] = normal(N, D, 1, 1).to(type)
        state["f"] = (normal(K, D, 1, 1) * (2.0 / math.sqrt(D))).to(type)
        state["b"] = 0.5 * normal(K) if case["bias"] else None
        labels = torch.randint(1, K + 1, (N,), generator=r, device="cuda").float()
        state["weights"] = None
        if case["skipped"]:
            labels = labels * (uniform(0.0, 1.0, N) < 0.9)
            state["weights"] = uniform(0.5, 1.5, N)
        state["labels"] = labels
    else:
        # a momentum: a few strong directions over noise
        n, rows, cols = case["count"], case["rows"], case["cols"]
        rank = max(1, min(rows, cols) // 8)
        strong = torch.bmm(normal(n, rows, rank) * torch.linspace(1.0, 0.05, rank, device="cuda"), normal(n, rank, cols))
        state["x"] = 1e-3 * (strong / math.sqrt(rank) + 0.3 * normal(n, rows, cols))
    return state


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    family = state["case"]["family"]
    return _run_lnorm(state) if family == "lnorm" else _run_fcloss(state) if family == "fcloss" else _run_ortho(state)


def _run_lnorm(s):
    both = s["case"]["what"] == "both"
    if own:
        from matconvnet_amd import capi
        y, moments = capi.lnorm_forward(s["x"], s["g"], s["b"], EPSILON)
        if not both:
            return {"y": y}
        dzdx, dzdg, dzdb = capi.lnorm_backward(s["x"], s["g"], s["dzdy"], EPSILON, moments=moments)
        return {"y": y, "dzdx": dzdx, "dzdg": dzdg, "dzdb": dzdb}
    x, g, b = s["x"].float(), s["g"].view(1, -1, 1, 1), s["b"].view(1, -1, 1, 1)
    centred = x - x.mean(dim=1, keepdim=True)
    sigma = torch.sqrt(centred.square().mean(dim=1, keepdim=True) + EPSILON)
    xh = centred / sigma
    y = (xh * g + b).to(s["x"].dtype)
    if not both:
        return {"y": y}
    dzdy = s["dzdy"].float()
    a = dzdy * g
    dzdx = (a - a.mean(dim=1, keepdim=True) - xh * (a * xh).mean(dim=1, keepdim=True)) / sigma
    return {"y": y, "dzdx": dzdx.to(s["x"].dtype), "dzdg": (dzdy * xh).sum(dim=(0, 2, 3)), "dzdb": dzdy.sum(dim=(0, 2, 3))}


def _run_fcloss(s):
    step = s["case"]["what"] == "step"
    if own:
        from matconvnet_amd import capi
        y, log_sums = capi.fcloss_forward(s["x"], s["f"], s["b"], s["labels"], instance_weights=s["weights"])
        if not step:
            return {"y": y, "log_sums": log_sums}
        dzdx, dzdf, dzdb = capi.fcloss_backward(s["x"], s["f"], s["b"], s["labels"], 1.0, instance_weights=s["weights"], log_sums=log_sums)
        return {"y": y, "log_sums": log_sums, "dzdx": dzdx, "dzdf": dzdf, "dzdb": dzdb}
    N = s["case"]["N"]
    x, f = s["x"].view(N, -1).float(), s["f"].view(s["case"]["K"], -1).float()
    z = x @ f.t()
    if s["b"] is not None:
        z = z + s["b"]
    w = (s["labels"] != 0).float()
    if s["weights"] is not None:
        w = w * s["weights"]
    at = (s["labels"].long() - 1).clamp(min=0).view(N, 1)
    most = z.max(dim=1, keepdim=True).values
    p = torch.exp(z - most)
    total = p.sum(dim=1, keepdim=True)
    log_sums = (most + torch.log(total)).view(N)
    y = ((w * (log_sums - z.gather(1, at).view(N))).double().sum() / N).float().view(1)
    if not step:
        return {"y": y, "log_sums": log_sums}
    p /= total
    p.scatter_add_(1, at, torch.full_like(total, -1.0))
    p *= (w / N).view(N, 1)
    dzdx = (p @ f).to(s["x"].dtype).view(s["x"].shape)
    dzdf = (p.t() @ x).to(s["f"].dtype).view(s["f"].shape)
    return {"y": y, "log_sums": log_sums, "dzdx": dzdx, "dzdf": dzdf, "dzdb": p.sum(dim=0)}


def _run_ortho(s):
    if own:
        from matconvnet_amd import capi
        return capi.orthogonalise(s["x"], steps=STEPS)
    tall = s["case"]["rows"] > s["case"]["cols"]
    x = s["x"].transpose(1, 2) if tall else s["x"]
    x = x / x.double().square().sum(dim=(1, 2), keepdim=True).sqrt().float()
    for _ in range(STEPS):
        g = torch.bmm(x, x.transpose(1, 2))
        x = A * x + torch.bmm(B * g + C * torch.bmm(g, g), x)
    return (x.transpose(1, 2) if tall else x).contiguous()


# ------------------------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["family"] == "lnorm":
        n, size = case["H"] * case["W"] * case["C"] * case["N"], _TYPES[case["type"]].itemsize
        return {"bytes": n * size * (2 if case["what"] == "forward" else 4), "flops": n * (8 if case["what"] == "forward" else 20)}
    if case["family"] == "fcloss":
        D, K, N, size = case["D"], case["K"], case["N"], _TYPES[case["type"]].itemsize
        step = case["what"] == "step"
        return {"bytes": (N + K) * D * size * (2 if step else 1), "flops": 2 * N * D * K * (3 if step else 1)}
    m, n = min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # (two of the three products are symmetric: half of each is enough)
    return {"bytes": 8 * m * n * case["count"], "flops": STEPS * case["count"] * (3 * m * m * n + m * m * m)}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["family"] == "lnorm":
            return _exact_lnorm(case, s)
        return _exact_fcloss(case, s) if case["family"] == "fcloss" else _exact_ortho(case, s)


def _exact_lnorm(case, s):
    """Rows of channels; the derivative by the Jacobian of a normalised row, (I - (1 1' + xh xh')/C)/sigma."""
    C = case["C"]
    rows = lambda t: t.double().permute(0, 2, 3, 1).reshape(-1, C)
    back = lambda t: t.view(case["N"], case["W"], case["H"], C).permute(0, 3, 1, 2).contiguous()
    x, g, b = rows(s["x"]), s["g"].double(), s["b"].double()
    sigma = torch.sqrt(x.var(dim=1, unbiased=False, keepdim=True) + EPSILON)
    xh = (x - x.mean(dim=1, keepdim=True)) / sigma
    out = {"y": back(xh * g + b)}
    if case["what"] == "both":
        d = rows(s["dzdy"])
        v = d * g
        out["dzdx"] = back((v - (v.sum(dim=1, keepdim=True) + xh * (v * xh).sum(dim=1, keepdim=True)) / C) / sigma)
        out["dzdg"], out["dzdb"] = (d * xh).sum(dim=0), d.sum(dim=0)
    return out


def _exact_fcloss(case, s):
    N, K = case["N"], case["K"]
    x, f = s["x"].double().view(N, -1), s["f"].double().view(K, -1)
    z = torch.mm(x, f.t())
    if s["b"] is not None:
        z += s["b"].double()
    log_sums = torch.logsumexp(z, dim=1)
    labelled = s["labels"] > 0
    w = labelled.double() if s["weights"] is None else labelled.double() * s["weights"].double()
    n, at = torch.arange(N, device=z.device), torch.where(labelled, s["labels"] - 1, 0.0).long()
    out = {"y": (w * (log_sums - z[n, at])).sum().view(1) / N, "log_sums": log_sums}
    if case["what"] == "step":
        z.sub_(log_sums[:, None]).exp_()
        z[n, at] -= 1.0
        z.mul_(w[:, None] / N)
        out["dzdx"], out["dzdf"] = torch.mm(z, f).view(s["x"].shape), torch.mm(z.t(), x).view(s["f"].shape)
        out["dzdb"] = z.sum(dim=0)
    return out


def _exact_ortho(case, s):
    """X <- P(X X') X with the polynomial formed as a matrix, on whichever side is shorter."""
    tall = case["rows"] > case["cols"]
    out = []
    for g in s["x"].double():
        x = g / torch.linalg.norm(g)
        m = min(x.shape)
        for _ in range(STEPS):
            gram = x.t() @ x if tall else x @ x.t()
            p = (C * gram + B * torch.eye(m, dtype=torch.float64, device=x.device)) @ gram
            p.diagonal().add_(A)
            x = x @ p if tall else p @ x
        out.append(x)
    return torch.stack(out)
