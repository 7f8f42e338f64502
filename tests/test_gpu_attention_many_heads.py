"""Attention of so many heads that the rows of one tile, position by position, would lie more than 2^31 bytes apart."""
import pytest
import torch

from tests.test_gpu_attention import Want, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [False, True])
def test_a_tile_of_positions_far_apart(capi, causal):
    """70 positions of 70000 heads of 128 in single precision: 35 MB from position to position, 63 times that from a tile's first row to its last"""
    n, heads, D = 70, 70000, 128
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("not enough memory")
    r = torch.Generator(device="cuda").manual_seed(3)
    q, k, v, dy = [torch.randn(n, heads, D, generator=r, device="cuda") for _ in range(4)]
    how = dict(causal=causal)
    y, sums = capi.attention_forward(q, k, v, **how)
    dq, dk, dv = capi.attention_backward(q, k, v, y, sums, dy, **how)
    some = torch.tensor([0, 1, 33333, 66999, heads - 1], device="cuda")
    w = Want(*[t[:, some].contiguous() for t in (q, k, v, dy)], [(n, n)], causal)
    for name, t in (("o", y), ("dq", dq), ("dk", dk), ("dv", dv)):
        near(t[:, some], getattr(w, name), getattr(w, name + "_off"), name)
    near(sums[:, some], w.sums, w.sums_off, "log sums")
