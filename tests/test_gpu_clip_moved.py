"""Lists of gradients whose memory has been exchanged since they were made."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gradients_and_outputs_that_moved(capi):
    r = torch.Generator(device="cuda").manual_seed(2)
    normal = lambda *s: torch.randn(s, generator=r, device="cuda")
    a, b = normal(1000), normal(20, 30)
    for separate in (False, True):
        outs = [torch.empty_like(a), torch.empty_like(b)] if separate else None
        plan = capi.GradientList([a, b], outs)
        capi.clip_gradients(plan, 1e9)
        for how in ("data", "set_"):
            old, new = a.detach(), 3 * normal(1000)
            kept, want = old.clone(), new.clone()
            if how == "data":
                a.data = new
            else:
                a.set_(new)
            norm = float(torch.cat([want, b.reshape(-1)]).double().norm())
            assert abs(float(capi.gradient_norm(plan)) - norm) <= 1e-6 * norm
            got = float(capi.clip_gradients(plan, 0.5 * norm))
            assert abs(got - norm) <= 1e-6 * norm
            torch.testing.assert_close((outs or [a])[0], 0.5 * want, rtol=1e-6, atol=0.0)
            if separate:
                assert torch.equal(a, want)
            assert torch.equal(old, kept)       # (what is the tensor's no longer is left alone)
        if separate:
            was = outs[1].detach()
            outs[1].data = torch.empty_like(b)
            kept = was.clone()
            capi.clip_gradients(plan, 1e9)
            assert torch.equal(outs[1], b) and torch.equal(was, kept)
    c = torch.zeros(1000, device="cuda")
    plan = capi.GradientList([a, c])
    c.data = a.data
    with pytest.raises(ValueError):
        capi.clip_gradients(plan, 1.0)
