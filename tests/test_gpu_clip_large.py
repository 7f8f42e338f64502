"""A tensor of more than 2^31 values, beside others: norm and clipped values.  The norm is a sum of squares in double, 2^-52 a step and off by less
than 2^-23 in all, rounded once (2^-24); a clipped value is a product in double, rounded once: 2^-8 of itself in bfloat16."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_more_values_than_31_bits_count(capi):
    n = 2 ** 31 + 2 ** 13 + 5
    big = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    values = torch.tensor([0.5, -1.0, 2.0, 0.25, -0.125, 1.5, 3.0], device="cuda").bfloat16()
    whole = n // 7 * 7
    big[:whole].view(-1, 7).copy_(values)
    big[whole:].copy_(values[:n - whole])
    small = torch.full((3, 1001), 2.0, device="cuda")
    squares = values.double().square()
    total = float(squares.sum()) * (n // 7) + float(squares[:n - whole].sum()) + 4.0 * small.numel()
    norm = capi.gradient_norm([big, small])
    assert abs(float(norm) - total ** 0.5) <= 2.0 ** -23 * total ** 0.5
    most = 1000.0
    again = capi.clip_gradients([big, small], most)
    assert float(again) == float(norm)
    want = values.double() * (most / total ** 0.5)
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -22 * want.abs()
    # ends, both sides of the borders between what one entry of a table holds, and everything in steps
    for at in (0, 2 ** 30 // 7 * 7 - 70, 2 ** 31 // 7 * 7 - 70, whole - 700):
        piece = big[at:at + 140].view(-1, 7).double()
        assert bool(((piece - want).abs() <= bound).all())
    rounded = big[:7].clone()
    for at in range(0, whole, 7 * 2 ** 26):
        piece = big[at:min(whole, at + 7 * 2 ** 26)].view(-1, 7)
        assert bool((piece == rounded).all())
    assert torch.equal(big[whole:], rounded[:n - whole])
    f = most / total ** 0.5
    assert float((small.double() - 2.0 * f).abs().max()) <= 2.0 * f * (2.0 ** -24 + 2.0 ** -22)


@pytest.mark.parametrize("count", [31, 32, 33, 163, 164, 165, 328, 329, 500])
def test_as_many_tensors_as_tables_hold_and_more(capi, count):
    r = torch.Generator(device="cuda")
    r.manual_seed(count)
    ders = [torch.randn((1 + 37 * i % 9001,), generator=r, device="cuda") for i in range(count)]
    total = sum(float(d.double().square().sum()) for d in ders) ** 0.5
    outs = [torch.empty_like(d) for d in ders]
    norm = capi.clip_gradients(capi.GradientList(ders, outs), 0.5 * total)
    assert abs(float(norm) - total) <= 2.0 ** -23 * total
    for d, y in zip(ders, outs):
        assert float((y.double() - 0.5 * d.double()).abs().max()) <= float(d.abs().max()) * 0.5 * (2.0 ** -24 + 2.0 ** -22)
