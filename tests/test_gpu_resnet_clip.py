"""ResNet-50's training step with clipped gradients, eagerly and replayed from a graph."""
import numpy as np
import pytest

from tests.util import bits_equal

pytestmark = pytest.mark.gpu
N, S, CLASSES = 4, 64, 40
LR, MOMENTUM, DECAY = 0.002, 0.9, 1e-4


def names(net):
    out = [("stem." + k, "stem.d" + k) for k in "fgb"]
    for i in range(net.units):
        for k in ("f1", "f2", "f3", "g1", "g2", "g3", "b1", "b2", "b3") + (("fs", "gs", "bs") if i in (0, 3, 7, 13) else ()):
            out.append(("unit%d.%s" % (i, k), "unit%d.d%s" % (i, k)))
    return out + [("fc.f", "fc.df"), ("fc.b", "fc.db")]


def start(net, seed=3):
    r = np.random.default_rng(seed)
    net.set("input", np.asfortranarray(r.standard_normal((S, S, 3, N), dtype=np.float32)))
    net.set("labels", np.asfortranarray(r.integers(1, CLASSES + 1, (1, 1, 1, N)).astype(np.float32)))


def step(net):
    net.forward()
    net.loss_derivative()
    net.backward()
    net.sgd_step(LR, MOMENTUM, DECAY)


def test_step_with_clipped_gradients(vl):
    net = vl.ResNet50(N=N, image_size=S, classes=CLASSES, seed=11)
    try:
        start(net)
        all_names = names(net)
        assert net.parameters == sum(net.get(v).size for v, _ in all_names)
        step(net)   # (a momentum to start from)
        for share in (0.25, 4.0):
            before = {v: (net.get(v), net.get("momentum." + v)) for v, _ in all_names}
            net.forward()
            net.loss_derivative()
            net.backward()
            ders = {v: net.get(d) for v, d in all_names}
            norm = np.sqrt(sum((d.astype(np.float64) ** 2).sum() for d in ders.values()))
            net.set_clip(share * norm)
            net.sgd_step(LR, MOMENTUM, DECAY)
            assert abs(float(net.get("gradientNorm").ravel()[0]) - norm) <= 2.0 ** -23 * norm
            factor = min(1.0, share)
            for v, _ in all_names:
                value, state = (t.astype(np.float64) for t in before[v])
                d = ders[v].astype(np.float64)
                want = MOMENTUM * state - (factor * d + DECAY * value)
                # the factor's rounding and four of the solver's, of the magnitudes' sum
                size = MOMENTUM * np.abs(state) + factor * np.abs(d) + DECAY * np.abs(value)
                assert (np.abs(net.get("momentum." + v) - want) <= 2.0 ** -21 * size + 1e-37).all(), v
                assert bits_equal(ders[v], net.get(dict(all_names)[v])), v   # (the derivatives stay as they are)
        net.set_clip(0.0)
        with pytest.raises(vl.VlError):
            net.set_clip(-1.0)
    finally:
        net.close()


def test_clipped_steps_from_a_graph(vl):
    import torch
    stream = torch.cuda.Stream()
    seen = {}
    with torch.cuda.stream(stream):
        for mode in ("eager", "graph"):
            net = vl.ResNet50(N=N, image_size=S, classes=CLASSES, seed=5)
            try:
                start(net)
                net.set_clip(0.5)
                step(net)
                if mode == "graph":
                    net.loss_derivative()
                    net.capture(True, LR, MOMENTUM, DECAY)
                out = []
                for i in range(3):
                    start(net, i)
                    if mode == "graph":
                        net.replay()
                    else:
                        net.forward()
                        net.backward()
                        net.sgd_step(LR, MOMENTUM, DECAY)
                    out.append({k: net.get(k) for k in ("gradientNorm", "stem.f", "unit7.f2", "momentum.fc.f")})
                seen[mode] = out
            finally:
                net.close()
    for a, b in zip(seen["eager"], seen["graph"]):
        for k in a:
            assert np.isfinite(a[k]).all() and bits_equal(a[k], b[k]), k
    assert float(seen["eager"][0]["gradientNorm"].ravel()[0]) > 0.5
