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


# ---- gates far open and far closed ----


def _logits(dtype):
    """Logits over the range where the sigmoid and one minus it are normal numbers of FP32."""
    top = 85.0
    g = torch.cat([torch.linspace(-top, top, 4001), torch.linspace(-8, 8, 1001), torch.tensor([0.0, -0.0, 1e-30])])
    return g[:g.numel() // 8 * 8].to(dtype).view(-1, 8).cuda()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["full", "channel", "row"])
def test_gates_far_open_and_closed(kind, dtype):
    """Each value of s and s (1 - s) to FP32's precision, however large the logit: with d of ones and no eps the
    update is the sigmoid itself, and the logit's gradient its slope."""
    logits = _logits(dtype)
    c = 8
    if kind == "channel":  # a call with a few rows for each eight of them
        calls = [(g.contiguous(), 3) for g in logits[::7]]
    elif kind == "row":
        calls = [(logits.reshape(-1, 1), logits.numel())]
    else:
        calls = [(logits, logits.shape[0])]
    # The exponential's argument to 2^-24 of it in two steps (16-bit rows: one, |g| 2^-24 <= 85 x 2^-24), the exponential
    # and the reciprocal of 1 ulp (2^-23) each, the reciprocal square root likewise, and eight roundings.
    rel = (8 + 1 + 2 * 3) * 2.0 ** -24 + (0 if dtype is F32 else 85 * 2.0 ** -24)
    one = torch.ones(c, device="cuda")
    for g, r in calls:
        x, dd = torch.zeros(r, c, dtype=dtype, device="cuda"), torch.ones(r, c, dtype=dtype, device="cuda")
        wide = d(g).expand(r, c)
        s, rest = torch.sigmoid(wide), torch.sigmoid(-wide)
        y, _ = ops.residual_norm(x, dd, one, g, eps=0.0)
        assert_within(y, s, rel * s)
        got = ops.residual_norm_gradient(x, dd, one, g, None, None, torch.ones_like(x), None, eps=0.0)[2]
        want = s * rest
        want = want.sum(0) if kind == "channel" else want.sum(1, keepdim=True) if kind == "row" else want
        # (1 - s is one more product of the same parts, and sums of up to eight equal terms are exact or off by a rounding)
        assert_within(got, want, (2 * rel + 8 * 2.0 ** -24) * want)
