"""GPU tests of the residual norm on outputs in place of inputs at every width's kernel, gates that are a column of a wider
array, and gradients in views of any alignment."""

import ctypes

import pytest
import torch

from _node_reference import Norm, assert_within
from symmetrix import _native
from symmetrix import node_ops as ops
from test_node_ops_gpu import BF16, F16, F32, _norm_inputs, _normal, _view, gen  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

WIDTHS = [5, 100, 130, 511, 777, 1001, 1500, 3001, 5003, 9999]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("c", WIDTHS)
def test_in_place(gen, c, dtype):  # noqa: F811
    """y over x, and dx over grad_y, as the C header allows."""
    r = 700
    x, dd, post, g, scale, nxt = _norm_inputs(gen, r, c, "row", dtype)
    gy, gh = _normal(gen, r, c, dtype=dtype), _normal(gen, r, c, dtype=dtype)
    stream = torch.cuda.current_stream().cuda_stream
    want = ops.residual_norm_gradient(x, dd, post, g, scale, nxt, gy, gh)
    inputs = ops._norm_inputs(x, dd, post, g, scale, nxt, 1e-6)
    size = _native.lib.smx_residual_norm_gradient_workspace(r, c)
    room = torch.empty(size, dtype=torch.uint8, device="cuda")
    a = _native.SmxResidualNormGradientArgs(_native.SmxResidualNormArgs(*inputs), gy.data_ptr(), c, gh.data_ptr(), c,
                                            gy.data_ptr(), c)
    a.workspace, a.workspace_bytes = room.data_ptr(), size
    _native.check(_native.lib.smx_residual_norm_gradient(ctypes.byref(a), stream))
    assert torch.equal(gy, want[0])
    y, h = ops.residual_norm(x, dd, post, g, scale, nxt)
    h2 = torch.empty_like(h)
    f = _native.SmxResidualNormArgs(*inputs, x.data_ptr(), c, h2.data_ptr(), c, None)
    _native.check(_native.lib.smx_residual_norm(ctypes.byref(f), stream))
    assert torch.equal(x, y) and torch.equal(h2, h)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("offset, more", [(0, 3), (1, 0), (5, 8)])
@pytest.mark.parametrize("c", [7, 130, 999, 2050])
def test_views(gen, c, offset, more, dtype):  # noqa: F811
    r = 37
    x, dd, post, _, scale, nxt = _norm_inputs(gen, r, c, "none", dtype)
    g = _normal(gen, r, 9, dtype=dtype)[:, 4:5]
    gy, gh = _normal(gen, r, c, dtype=dtype), _normal(gen, r, c, dtype=dtype)
    f = Norm(x, dd, post, g, scale, nxt, 1e-6)
    x, dd, gy, gh = (_view(t, offset, more) for t in (x, dd, gy, gh))
    y, h = ops.residual_norm(x, dd, post, g, scale, nxt)
    assert_within(y, f.y, f.y_bound)
    assert_within(h, f.h, f.h_bound)
    got = ops.residual_norm_gradient(x, dd, post, g, scale, nxt, gy, gh)
    want, bound = f.backward(gy, gh)
    for name, t in zip(("x", "d", "gate", "post", "scale", "next"), got):
        assert_within(t, want[name], bound[name])
