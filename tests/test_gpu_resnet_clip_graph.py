"""A captured training step and a largest norm of the gradients that changes behind it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_another_norm_drops_the_graph(vl):
    import torch
    rates = (0.002, 0.9, 1e-4)
    with torch.cuda.stream(torch.cuda.Stream()):
        net = vl.ResNet50(N=4, image_size=64, classes=40, seed=5)
        try:
            r = np.random.default_rng(0)
            net.set("input", np.asfortranarray(r.standard_normal((64, 64, 3, 4), dtype=np.float32)))
            net.set("labels", np.asfortranarray(r.integers(1, 41, (1, 1, 1, 4)).astype(np.float32)))
            net.set_clip(0.5)
            net.forward()
            net.loss_derivative()
            net.backward()
            net.sgd_step(*rates)
            net.capture(True, *rates)
            net.replay()
            net.set_clip(0.5)      # (as it was)
            net.replay()
            for other in (0.25, 0.0):
                net.set_clip(other)
                with pytest.raises(vl.VlError) as e:
                    net.replay()
                assert "nothing has been captured" in e.value.message
                net.capture(True, *rates)
                net.replay()
            assert np.isfinite(net.get("stem.f")).all()
        finally:
            net.close()
