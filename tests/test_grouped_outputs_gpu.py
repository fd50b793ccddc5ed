"""GPU tests that the products by type write every output: at the C boundary, where outputs are the caller's and hold NaN before
the call, at sizes that reach each of the kernels' cuts."""

import math

import pytest
import torch

from symmetrix import node_ops as ops
from symmetrix._native import lib
from test_grouped_cuts_gpu import FEW, TILES
from test_grouped_gpu import BF16, F16, F32, _check, _normal, _types, gen  # noqa: F401 (gen: a fixture)

pytestmark = pytest.mark.gpu

CODES = {F32: 0, BF16: 1, F16: 2}
# a type's tiles fill the card: nothing is cut, and no workspace is given
LARGE = [(700, 1, 4096, 4104, "any"), (1200, 2, 4104, 4096, "outside")]


def _filled(*shape, dtype):
    return torch.full(shape, math.nan, dtype=dtype, device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, v, k, n, kind", FEW + TILES + LARGE)
def test_every_output_is_written(gen, rows, v, k, n, kind, dtype):  # noqa: F811
    """And is what the Python call gives, which the other tests hold against float64."""
    z = _types(gen, rows, v, kind)
    x, w, grad = _normal(gen, rows, k, dtype=dtype), _normal(gen, v, n, k, dtype=dtype), _normal(gen, rows, n, dtype=dtype)
    groups = ops.group_rows(z, v)
    y, dx, dw = _filled(rows, n, dtype=dtype), _filled(rows, k, dtype=dtype), _filled(v, n, k, dtype=F32)
    code, plan, s = CODES[dtype], groups._room.data_ptr(), torch.cuda.current_stream().cuda_stream
    size = lib.smx_grouped_linear_by_weights_workspace(rows, v, k, n)
    room = _filled(max(4, size // 4), dtype=F32)
    assert lib.smx_grouped_linear(x.data_ptr(), k, code, w.data_ptr(), k, n * k, plan, rows, v, k, n, code, y.data_ptr(), n, s) == 0
    assert lib.smx_grouped_linear_by_rows(grad.data_ptr(), n, code, w.data_ptr(), k, n * k, plan, rows, v, k, n, code, dx.data_ptr(),
                                          k, s) == 0
    assert lib.smx_grouped_linear_by_weights(grad.data_ptr(), n, x.data_ptr(), k, code, plan, rows, v, k, n, 0, dw.data_ptr(), k,
                                             n * k, room.data_ptr(), size, s) == 0
    for got in (y, dx, dw):
        assert torch.isfinite(got).all()
    assert torch.equal(y, ops.grouped_linear(x, w, groups))
    for a, b in zip((dx, dw), ops.grouped_linear_gradient(grad, x, w, groups)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows, v, k, n, kind", LARGE)
def test_types_that_fill_the_card(gen, rows, v, k, n, kind, dtype):  # noqa: F811
    z = _types(gen, rows, v, kind)
    assert lib.smx_grouped_linear_by_weights_workspace(rows, v, k, n) == 0
    _check(z, v, _normal(gen, rows, k, dtype=dtype), _normal(gen, v, n, k, dtype=dtype), _normal(gen, rows, n, dtype=dtype))
