"""Attention of values that are not finite: what it costs where they are seen anyway."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def microseconds(f):
    f()
    torch.cuda.synchronize()
    best = math.inf
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, 1e3 * a.elapsed_time(b))
    return best


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_is_seen_is_not_added_up_anew(capi, dtype):
    """One value, key or query that is not finite and that (nearly) all rows or keys see: a hundred times the time where each of them were added
    up again one by one; ten times is allowed (a look at the rows around the mask's edge)"""
    n, heads = 4096, 4
    r = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, dy = [torch.randn(n, h, 128, generator=r, device="cuda").to(dtype) for h in (heads, 1, 1, heads)]
    y, sums = capi.attention_forward(q, k, v, causal=True)
    # a value of the second half of the first tile of 64 keys
    v2 = v.clone()
    v2[40, :, 3] = math.nan
    forward = lambda v: capi.attention_forward(q, k, v, causal=True)
    got = forward(v2)[0]
    assert bool(torch.isnan(got[40:, :, 3]).all()) and torch.equal(got[:32], y[:32])
    assert microseconds(lambda: forward(v2)) <= 10 * microseconds(lambda: forward(v))
    # a key there, to dq (of the log sums without it)
    k2 = k.clone()
    k2[40, :, 3] = math.nan
    backward = lambda q, k, *want: capi.attention_backward(q, k, v, y, sums, dy, causal=True, want=want)
    assert bool(torch.isnan(backward(q, k2, True, False, False)[0][40:, :, 3]).all())
    assert microseconds(lambda: backward(q, k2, True, False, False)) <= 10 * microseconds(lambda: backward(q, k, True, False, False))
    # the last query of the group's second head, to dk and dv
    q2 = q.clone()
    q2[n - 1, 1] = math.nan
    _, dk, dv = backward(q2, k, False, True, True)
    assert bool(torch.isnan(dk).all()) and bool(torch.isnan(dv).all())
    assert microseconds(lambda: backward(q2, k, False, True, True)) <= 10 * microseconds(lambda: backward(q, k, False, True, True))
