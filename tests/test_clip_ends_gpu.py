"""GPU tests of clipping at the ends of FP32's range: subnormal values, factors far above and far below one, and an infinite
norm that is not clipped, against the definition in float64."""

import math

import pytest
import torch

from _node_reference import assert_within, d
from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LARGEST = torch.finfo(F32).max


def _small(power, count=50):
    """Whole multiples of 2^power on both sides of zero, more than a lane takes at once and no whole number of sixteen bytes."""
    return (torch.arange(-count, count + 1, device="cuda").double() * 2.0 ** power).float()


def _clipped(t, most, scale, out):
    """(norm, values) in place (out None) or to tensors of type `out`"""
    held = t.clone()
    if out is None:
        return ops.clip_gradients([held], most, scale=scale), held
    to = torch.full_like(held, math.nan, dtype=out)
    norm = ops.clip_gradients([held], most, scale=scale, out=[to])
    assert torch.equal(held.view(torch.int32), t.view(torch.int32))  # (bits: a NaN is one)
    return norm, to


@pytest.mark.parametrize("count", [1, 50, 20000])
@pytest.mark.parametrize("out", [None, F32], ids=["in place", "out"])
@pytest.mark.parametrize("scale", [1.0, 2.0, 3.0, 0.5, 0.75, 2.0 ** 100, 2.0 ** 127, LARGEST])
def test_factors_that_are_scales(scale, out, count):
    """A norm below max_norm: every value times the scale, rounded once, subnormal values among them.  (The products have 48
    bits at most: exact in float64, which rounds them to FP32 once.)"""
    t = torch.cat([_small(-149, count), torch.tensor([2.0 ** -126, -3e-39, 0.0], device="cuda")])
    norm, got = _clipped(t, 2.0 ** 20, scale, out)
    want = t.double() * torch.tensor(scale).double().item()
    assert torch.equal(got, want.float()) and norm.item() <= 2.0 ** 20
    assert torch.equal(torch.signbit(got), torch.signbit(want))


@pytest.mark.parametrize("out", [None, F32, BF16, F16], ids=["in place", "f32", "bf16", "f16"])
@pytest.mark.parametrize("most, scale", [(2.0 ** -25, 1.0), (1e-10, 1e-30), (2.0 ** -25, 2.0 ** -20), (2.0 ** 10, 2.0 ** -149), (1.0, 1.0)])
def test_factors_below_subnormal_numbers(most, scale, out):
    """Values next to FP32's largest, whose factor is below its least number and whose products are normal numbers."""
    t = torch.cat([torch.full((1000,), 3e38, device="cuda"), torch.full((37,), -LARGEST, device="cuda"), _small(100), _small(-149)])
    size = d(t).square().sum().sqrt().item()
    norm, got = _clipped(t, most, scale, out)
    most, scale = (torch.tensor(v).double().item() for v in (most, scale))  # as FP32 has them
    total = scale * size
    factor = scale if total <= most else most / size
    if total <= LARGEST:
        # (rounded once; the sum of squares is off by far less)
        assert abs(norm.item() - total) <= (2.0 ** -24 + 2.0 ** -40) * total + 2.0 ** -150
    # the factor's significand and its product are rounded to FP32, 2^-24 each, and the result to its type
    want = d(t) * factor
    assert_within(got, want, 2.0001 * 2.0 ** -24 * want.abs())


@pytest.mark.parametrize("out", [None, F32], ids=["in place", "out"])
def test_large_scales_that_are_clipped(out):
    """A scale of 2^127 on values whose norm is clipped: the factor is between the scale and one."""
    t = torch.randn(1000, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 2.0 ** -100
    size = d(t).square().sum().sqrt().item()
    norm, got = _clipped(t, 0.5, 2.0 ** 127, out)
    assert abs(norm.item() - size * 2.0 ** 127) <= (2.0 ** -24 + 2.0 ** -40) * size * 2.0 ** 127
    want = d(t) * 0.5 / size
    assert_within(got, want, 2.0001 * 2.0 ** -24 * want.abs())


@pytest.mark.parametrize("out", [None, F32], ids=["in place", "out"])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_no_clipping_of_an_infinite_norm(scale, out):
    """max_norm infinite clips nothing, whatever the norm is; a NaN still makes all NaN."""
    t = torch.tensor([1.0, math.inf, -3.0, 0.0, -math.inf], device="cuda")
    norm, got = _clipped(t, math.inf, scale, out)
    assert norm.item() == math.inf and torch.equal(got, t * scale)
    t[2] = math.nan
    norm, got = _clipped(t, math.inf, scale, out)
    assert math.isnan(norm.item()) and torch.isnan(got).all()
