"""GPU tests of the products by type at the ends of their types' ranges, and with plans that are not theirs."""

import pytest
import torch

from _node_reference import assert_within, d
from symmetrix import node_ops as ops
from symmetrix._native import lib

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _three(x, w, grad):
    groups = ops.group_rows(torch.zeros(len(x), dtype=torch.int32, device="cuda"), 1)
    return [ops.grouped_linear(x, w[None], groups, F32), *ops.grouped_linear_gradient(grad, x, w[None], groups)]


@pytest.mark.parametrize("rows", [10, 700])
def test_subnormal_float16(rows):
    """FP16's subnormal numbers are numbers: whole multiples of 2^-24, whose products with whole numbers are exact."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randint(-9, 10, (rows, 64), generator=g, device="cuda") * 2.0 ** -24).to(F16)
    w = torch.randint(-3, 4, (40, 64), generator=g, device="cuda").to(F16)
    grad = torch.randint(-3, 4, (rows, 40), generator=g, device="cuda").to(F16)
    y, dx, dw = _three(x, w, grad)
    assert torch.equal(d(y), d(x) @ d(w).T) and torch.equal(d(dw[0]), d(grad).T @ d(x)) and d(x).abs().sum() > 0


@pytest.mark.parametrize("rows", [10, 700])
@pytest.mark.parametrize("power", [-120, -110, -104, -90])
def test_small_float32(rows, power):
    """Values whose last parts leave bf16's normal numbers: off by less than 2^-126 each, times the other operand."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, 64, generator=g, device="cuda") * 2.0 ** power
    w = torch.randn(40, 64, generator=g, device="cuda") * 2.0 ** 60
    y = _three(x, w, torch.randn(rows, 40, generator=g, device="cuda"))[0]
    want, size = d(x) @ d(w).T, d(x).abs() @ d(w).abs().T
    # (two of a value's parts may be below)
    assert_within(y, want, (64 + 24) * 2.0 ** -23 * size + 2 * 2.0 ** -126 * d(w).abs().sum(1))


@pytest.mark.parametrize("rows", [10, 700])
def test_large_float32(rows):
    """Values up to FP32's largest, which round to infinity in bf16, stay finite."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.where(torch.rand(rows, 64, generator=g, device="cuda") < 0.5, 1.0, -1.0) * torch.finfo(F32).max
    w = torch.randn(40, 64, generator=g, device="cuda") * 2.0 ** -20
    y = _three(x, w, torch.zeros(rows, 40, device="cuda"))[0]
    assert torch.isfinite(y).all()
    assert_within(y, d(x) @ d(w).T, (64 + 24) * 2.0 ** -23 * (d(x).abs() @ d(w).abs().T))


def test_outputs_beyond_the_type():
    x, w = torch.full((5, 64), 300.0, device="cuda", dtype=F16), torch.full((8, 64), 300.0, device="cuda", dtype=F16)
    groups = ops.group_rows(torch.zeros(5, dtype=torch.int32, device="cuda"), 1)
    assert torch.isinf(ops.grouped_linear(x, w[None], groups)).all()
    assert (ops.grouped_linear(x, w[None], groups, F32) == 64 * 300.0 ** 2).all()


def test_plans_of_other_rows():
    """With a plan of other rows or types nothing is read or written."""
    s = torch.cuda.current_stream().cuda_stream
    for rows, other, v in ((700, 600, 3), (700, 800, 3), (20, 30, 9), (20, 10, 9)):
        x, w = torch.randn(rows, 40, device="cuda"), torch.randn(v, 24, 40, device="cuda")
        grad = torch.randn(rows, 24, device="cuda")
        y, dx, dw = torch.full((rows, 24), 5.0, device="cuda"), torch.full((rows, 40), 5.0, device="cuda"), \
            torch.full((v, 24, 40), 5.0, device="cuda")
        size = lib.smx_grouped_linear_by_weights_workspace(rows, v, 40, 24)
        room = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
        for plan, kinds in ((ops.group_rows(torch.zeros(other, dtype=torch.int32, device="cuda"), v), v),
                            (ops.group_rows(torch.zeros(rows, dtype=torch.int32, device="cuda"), v + 1), v)):
            at = plan._room.data_ptr()
            assert lib.smx_grouped_linear(x.data_ptr(), 40, 0, w.data_ptr(), 40, 960, at, rows, kinds, 40, 24, 0, y.data_ptr(), 24, s) == 0
            assert lib.smx_grouped_linear_by_rows(grad.data_ptr(), 24, 0, w.data_ptr(), 40, 960, at, rows, kinds, 40, 24, 0,
                                                  dx.data_ptr(), 40, s) == 0
            assert lib.smx_grouped_linear_by_weights(grad.data_ptr(), 24, x.data_ptr(), 40, 0, at, rows, kinds, 40, 24, 0, dw.data_ptr(),
                                                     40, 960, room.data_ptr(), size, s) == 0
            torch.cuda.synchronize()
            assert (y == 5).all() and (dx == 5).all() and (dw == 5).all()
