"""GPU tests of what products by type keep of small FP32 values: their bf16 parts are multiples of 2^-133."""

import pytest
import torch

from _node_reference import d
from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [10, 700])
@pytest.mark.parametrize("power", [-149, -140, -133, -127, -120, -111])
def test_parts_of_small_values(rows, power):
    """One term, by a power of two: a value below 2^-110 is off by half a step of 2^-133 at most, and a larger one not at all (its
    24 bits are three parts')."""
    gen = torch.Generator(device="cuda").manual_seed(41)
    whole = torch.randint(-(1 << 23) + 1, 1 << 23, (rows, 1), generator=gen, device="cuda").double()
    groups = ops.group_rows(torch.zeros(rows, dtype=torch.int32, device="cuda"), 1)
    w = torch.full((1, 40, 1), 2.0 ** 100, device="cuda")
    for up, bound in ((power - 22, 2.0 ** -134), (-132, 0.0)):
        x = (whole * 2.0 ** up).float()
        grad = torch.zeros(rows, 40, device="cuda")
        grad[:, 7:8] = x
        y = ops.grouped_linear(x, w, groups)
        dx, dw = ops.grouped_linear_gradient(grad, torch.full_like(x, 2.0 ** 100), w, groups)
        for got in (y, dx):
            assert ((d(got) * 2.0 ** -100 - d(x)).abs() <= bound).all()
        # (a sum of as many terms: as many roundings of its partial sums)
        size = d(x).abs().sum()
        assert abs(d(dw)[0, 7, 0] * 2.0 ** -100 - d(x).sum()) <= rows * (bound + 2.0 ** -24 * size)
