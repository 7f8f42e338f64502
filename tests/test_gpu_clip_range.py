"""The solver's step with clipping where the factor is no number of single precision."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,most", [(1e25, 1e-20), (1e20, 1e-18), (1e30, 1.0)])
def test_factors_below_single_precision(capi, size, most):
    """state = -(factor der): one product in double, rounded once (2^-24), of a factor whose norm is off by 2^-40"""
    chunks = 3
    r = torch.Generator(device="cuda").manual_seed(1)
    der = size * torch.randn(chunks * capi.SGD_CHUNK, generator=r, device="cuda")
    value, state = torch.zeros_like(der), torch.zeros_like(der)
    table = torch.zeros(chunks, dtype=torch.int16, device="cuda")
    rates = torch.ones(1, 2, dtype=torch.float64, device="cuda")
    for scale in (1.0, -0.25):
        norm = abs(scale) * float(der.double().square().sum().sqrt())
        state.zero_()
        value.zero_()
        capi.sgd_momentum_clipped(value, state, der, table, rates, 0.5, 0.0, 0.9, most, der_scale=scale)
        want = -(scale * most / norm) * der.double()
        assert bool(((state.double() - want).abs() <= (2.0 ** -24 + 2.0 ** -40) * want.abs() + 2.0 ** -149).all())
        assert bool(((value.double() - 0.5 * want).abs() <= (2.0 ** -23 + 2.0 ** -40) * 0.5 * want.abs() + 2.0 ** -149).all())
