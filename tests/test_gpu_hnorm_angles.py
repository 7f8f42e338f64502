"""The cosines and sines that hnorm turns heads by, against double precision.

A pair (1, 0) becomes (cos, sin).  Each is off by two units in the last place of the sine's function (2^-22 of it), half a one of its correction and of
the product with 1 (2^-23): 2^-21 of itself together; the angle, a sum of `axes` products in double brought to revolutions by one more, by (axes + 3) 2^-53 of the
sum of magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("far", [0, 1000003])
@pytest.mark.parametrize("axes,pairs", [(1, 64), (3, 20), (1, 100), (5, 32)])     # (up to 3 axes and 64 pairs, and others: made on different ways)
def test_all_of_a_single_precision_sine(capi, axes, pairs, far):
    N = 700
    r = torch.Generator(device="cuda").manual_seed(axes + pairs)
    positions = torch.arange(N, device="cuda", dtype=torch.float64).view(N, 1) + far + torch.arange(axes, device="cuda", dtype=torch.float64) * 7
    frequencies = torch.rand(axes, pairs, generator=r, device="cuda", dtype=torch.float64) + 0.001
    frequencies[:, 0] = 1.0
    q = torch.zeros(N, 1, 2 * pairs, device="cuda")
    q[:, :, :pairs] = 1.0
    y, _ = capi.hnorm_forward(q, None, None, None, positions, frequencies, normalise=False)
    angle = positions @ frequencies
    off = (axes + 3) * 2.0 ** -53 * angle.abs()
    for got, want in ((y[:, 0, :pairs], torch.cos(angle)), (y[:, 0, pairs:], torch.sin(angle))):
        assert bool(((got.double() - want).abs() <= 2.0 ** -21 * want.abs() + 2 * off).all()), float(((got.double() - want).abs() / want.abs()).max())
    # ... and turned back
    dq, _, _, _ = capi.hnorm_backward(q, None, None, None, positions, frequencies, y, None, normalise=False)
    assert bool(((dq - q).abs() <= 2.0 ** -20).all())
