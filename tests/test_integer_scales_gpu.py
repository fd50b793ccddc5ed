"""GPU tests of integer products whose scales lie far apart: a product of both scales and the sum that is a number of the
outputs' type is one, whatever the sum times one scale alone would be."""

import math

import pytest
import torch

from _node_reference import assert_within, d
from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _integers(gen, rows, k, scales):
    values = torch.zeros(rows, -(-k // 128) * 128, dtype=torch.int8, device="cuda")
    values[:, :k] = torch.randint(-127, 128, (rows, k), generator=gen)
    return ops.IntegerValues(values, scales.to("cuda", F32), (rows, k))


def _want(a, b):
    """(sums of whole numbers below 2^53: exact on the card in float64)"""
    sums = torch.matmul(a.values.double(), b.values.double().T.contiguous())
    return (sums * a.scales.double()[:, None] * b.scales.double()[None]).cpu()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("m, n, k", [(3, 40, 200), (13, 37, 1000), (70, 50, 300), (300, 700, 128)])
def test_scales_far_apart(m, n, k, dtype):
    gen = torch.Generator().manual_seed(23)
    large, small = [2.0 ** 121, 1.7e36, 2.0 ** 100, 3.0], [2.0 ** -126, 3.1e-38, 2.0 ** -110, 0.3]
    for one, other in ((large, small), (small, large), (large + small, large + small)):
        a, b = (_integers(gen, r, k, torch.tensor([s[i % len(s)] for i in range(r)])) for r, s in ((m, one), (n, other)))
        # one rounding when the sum becomes FP32 and one at each scale
        want = _want(a, b)
        got = ops.integer_product(a, b, dtype)
        assert torch.isfinite(got).any()
        # (what lies next to the type's largest number may round to it or to infinity)
        most = torch.finfo(dtype).max
        clear = (want.abs() < most * (1 - 2.0 ** -20)) | (want.abs() > most * (1 + 2.0 ** -8))
        assert_within(torch.where(clear.cuda(), got, 0), torch.where(clear, want, 0), 3.0001 * 2.0 ** -24 * want.abs())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 4, 11, 90])
def test_rows_next_to_the_largest_number(m, dtype):
    """x next to FP32's largest number, through weights that bring it back: finite, though the sum times x's scale is not."""
    gen = torch.Generator().manual_seed(29)
    x = (torch.randn(m, 500, generator=gen).clamp(-3, 3) * 1e38).to("cuda", dtype)
    w = torch.randn(60, 500, generator=gen).cuda() * 2.0 ** -20
    for rows, weights in ((x, w), (w.to(dtype)[:m], x.float())):
        a, b = ops.quantize_integers(rows), ops.quantize_integers(weights)
        want = _want(a, b)
        assert want.abs().max() < 1e38
        got = ops.integer_linear(rows, b)
        assert torch.isfinite(got).all()
        assert_within(got, want, 3.0001 * 2.0 ** -24 * want.abs())


@pytest.mark.parametrize("m", [3, 90])
def test_scales_of_another_making(m):
    """Negative scales, zeros and such as are no numbers, on either side."""
    gen = torch.Generator().manual_seed(31)
    odd = torch.tensor([-2.0, 0.0, math.nan, math.inf, 1.0, -1e-30])
    one = torch.tensor([1.0, 3.0, -5.0, 0.25, 2.0, 8.0])
    for p, q in ((odd, one), (one, odd)):
        a, b = _integers(gen, m, 130, p.repeat(-(-m // 6))[:m]), _integers(gen, 66, 130, q.repeat(11))
        a.values[0] = 0  # (sums of zero: with a scale of infinity NaN)
        want = _want(a, b)
        assert_within(ops.integer_product(a, b), want, 3.0001 * 2.0 ** -24 * want.abs())
