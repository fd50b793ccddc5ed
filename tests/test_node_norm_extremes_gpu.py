"""GPU tests of the residual norm where single rows are infinite and where gates are far open or far closed."""

import math

import pytest
import torch

from _node_reference import Norm, assert_within, d
from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
IDS = ["f32", "bf16", "f16"]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("gate", ["none", "full", "channel", "row"])
@pytest.mark.parametrize("c, following", [(40, False), (40, True), (300, True), (999, False), (4100, True)])
def test_gradient_without_grad_h_of_infinite_rows(c, following, gate, dtype):
    """Without h's gradient, x and y do not enter any gradient: an infinity in x (or one whose square is)
    stays out of them."""
    g = torch.Generator(device="cuda").manual_seed(9)
    r = 7

    def n(*s, t=dtype):
        return torch.randn(*s, generator=g, device="cuda").to(t)
    x, dd, gy = n(r, c), n(r, c), n(r, c)
    post, scale, nxt = (1 + 0.3 * n(c, t=F32) for _ in range(3))
    shape = {"none": None, "full": (r, c), "channel": (c,), "row": (r, 1)}[gate]
    logits = None if shape is None else n(*shape)
    f = Norm(x, dd, post, logits, scale, nxt, 1e-6)
    want, bound = f.backward(gy, None)
    x[1, 3], x[2, 5] = math.inf, -math.inf
    x[4] = torch.finfo(dtype).max
    got = dict(zip(("x", "d", "gate", "post", "scale", "next"), ops.residual_norm_gradient(
        x, dd, post, logits, scale, nxt if following else None, gy, None)))
    assert torch.equal(got["x"], gy)
    for name in ("d", "gate", "post", "scale"):
        if got[name] is not None:
            assert_within(got[name], want[name], bound[name])
    assert got["next"] is None if not following else (got["next"] == 0).all()
