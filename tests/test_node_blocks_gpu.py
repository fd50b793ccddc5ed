"""GPU tests of the head built of the node operators (symmetrix.node_blocks): its gradients against a
plain float64 form of the same arithmetic, training on an evaluator's energies, and serving."""

import math

import pytest
import torch

from _node_reference import d, quantized
from symmetrix import node_blocks

pytestmark = pytest.mark.gpu


class _Product(torch.autograd.Function):
    """a @ b.T of 8-bit blocks in float64, each product's operands in blocks along its summed axis."""

    @staticmethod
    def forward(ctx, a, b):
        ctx.save_for_backward(a, b)
        return quantized(a)[0] @ quantized(b)[0].T

    @staticmethod
    def backward(ctx, g):
        a, b = ctx.saved_tensors
        return quantized(g)[0] @ quantized(b.T)[0].T, quantized(g.T)[0] @ quantized(a.T)[0].T


def _plain(model, p, types, desc):
    c = model.channels

    def norm(x, w):
        return x / torch.sqrt(x.pow(2).mean(1, keepdim=True) + model.eps) * w
    x = p["table"][types] * math.sqrt(c) + _Product.apply(desc, p["lift"])
    h = norm(x, p["before"])
    for k in range(len(model.weights)):
        both = _Product.apply(h, p["weights.%d" % k])
        x = x + p["scale.%d" % k] * torch.sigmoid(both[:, c:]) * norm(both[:, :c], p["post.%d" % k])
        h = norm(x, p["next.%d" % k])
    return h @ p["readout"] + p["shift"][types]


@pytest.mark.parametrize("channels, blocks", [(64, 1), (130, 2)])
def test_gradients(channels, blocks):
    torch.manual_seed(3)
    n = 90
    model = node_blocks.NodeBlocks(5, 24, channels, blocks).cuda()
    types = torch.randint(0, 5, (n,), device="cuda", dtype=torch.int32)
    desc, w = torch.randn(n, 24, device="cuda"), torch.randn(n, device="cuda")
    e = model(types, desc)
    (e * w).sum().backward()
    p = {k: d(v).requires_grad_() for k, v in model.named_parameters()}
    want = _plain(model, p, types.cpu().long(), d(desc))
    (want * d(w)).sum().backward()
    # An FP32 rounding (2^-20 with its sums) moves a value across the boundary of two 8-bit ones, 2^-4
    # apart, in 2^-16 of the cases: 2^-4 / 2^8 = 2^-12 of a product's norm, doubled by each of the few products after it
    bound = 2.0 ** -12 * 2 ** (2 * blocks + 2)
    assert (d(e) - want).norm() < bound * want.norm()
    for k, v in model.named_parameters():
        assert (d(v.grad) - p[k].grad).norm() <= bound * p[k].grad.norm(), k


def test_fit_and_serve():
    got = node_blocks.fit(steps=150, cells=2, report=None)
    assert got["trained"] < 0.5 * got["means"]
    # the served head's rows are brought to 8 bits from FP32 norms as the trained one's are
    assert abs(got["served"] - got["trained"]) < 0.02 * got["means"]


def test_served_types():
    torch.manual_seed(4)
    types = torch.randint(0, 5, (40,), device="cuda", dtype=torch.int32)
    desc = torch.randn(40, 24, device="cuda")
    for dtype, rel in ((torch.float32, 2.0 ** -8), (torch.bfloat16, 2.0 ** -5), (torch.float16, 2.0 ** -7)):
        model = node_blocks.NodeBlocks(5, 24, 128, 3, dtype).cuda()
        with torch.no_grad():
            want = model(types, desc)
            got = model.serve()(types, desc)
        # roundings of rows to the type, and of a few 8-bit values to their neighbours
        assert (got - want).norm() < rel * want.norm()
        one = model.serve()(types[:1], desc[:1])  # a single atom takes the kernels for few rows
        assert (one - got[:1]).abs().item() < rel * got.norm().item()
