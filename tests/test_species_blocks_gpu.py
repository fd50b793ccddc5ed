"""GPU tests of the operators of rows by type, clipping and integers as the head uses them together (symmetrix.node_blocks)."""

import copy
import math

import pytest
import torch

from symmetrix import node_blocks
from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu


def _data(n=300, v=6):
    g = torch.Generator(device="cuda").manual_seed(3)
    return (torch.randint(-1, v + 1, (n,), generator=g, device="cuda", dtype=torch.int32),
            torch.randn(n, 24, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda"))


def _by_hand(model, types, desc):
    """The head in float64, its weights by species."""
    p = {k: v.detach().double() for k, v in model.named_parameters()}
    there = (types >= 0) & (types < model.table.shape[0])
    z = torch.where(there, types, 0).long()
    c, eps = model.channels, model.eps

    def unit(x):
        return x / torch.sqrt(x.square().mean(1, keepdim=True) + eps)
    d = torch.where(there[:, None], desc.double(), 0)
    x = torch.where(there[:, None], p["table"][z] * math.sqrt(c), 0) + d @ p["lift"].T
    h = unit(x) * p["before"]
    for k in range(len(model.weights)):
        both = (p["weights.%d" % k][z] * h[:, None, :]).sum(2)
        both = torch.where(there[:, None], both, 0)
        x = x + p["scale.%d" % k] * torch.sigmoid(both[:, c:]) * p["post.%d" % k] * unit(both[:, :c])
        h = unit(x) * p["next.%d" % k]
    return torch.where(there, h @ p["readout"] + p["shift"][z], 0)


@pytest.mark.parametrize("form", ["blocks", "integers"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_head_by_species(dtype, form):
    torch.manual_seed(5)
    model = node_blocks.NodeBlocks(6, 24, 64, 2, dtype, by_species=True).cuda()
    types, desc, w = _data()
    want = _by_hand(model, types, desc)
    e = model(types, desc)
    # The descriptors' linear is in 8-bit blocks: values of four significant bits, 2^-4 each, of which a sum of 24 keeps about a
    # fifth (2^-4 / sqrt(24) of its terms' norm); two normed blocks pass it on.  8-bit integers are finer.
    size = want.square().mean().sqrt()
    assert (e - want).square().mean().sqrt() < 0.1 * size
    (e * w).sum().backward()
    absent = torch.ones(6, dtype=torch.bool, device="cuda")
    absent[types[(types >= 0) & (types < 6)].long()] = False
    for p in model.parameters():
        assert torch.isfinite(p.grad).all()
    for p in model.weights:
        assert p.grad.dtype is torch.float32 and not p.grad[absent].any()
    got = model.serve(form)(types, desc)
    assert (got - want).square().mean().sqrt() < 0.1 * size and (got[(types < 0) | (types >= 6)] == 0).all()


def test_a_training_step_in_a_graph():
    """Forward, backward, the gradients' clipping and a plain step, captured together and replayed: the same weights as
    the eager step's, with eager work on other data between the replays."""
    torch.manual_seed(7)
    model = node_blocks.NodeBlocks(6, 24, 64, 2, by_species=True).cuda()
    twin = copy.deepcopy(model)
    types, desc, target = _data(128)
    held = types.clone(), desc.clone(), target.clone()

    def step(model, types, desc, target):
        loss = (model(types, desc) - target).square().mean()
        grads = torch.autograd.grad(loss, list(model.parameters()))
        norm = ops.clip_gradients(grads, 0.01)
        with torch.no_grad():
            for p, g in zip(model.parameters(), grads):
                p -= g
        return norm
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    spare = copy.deepcopy(model)
    with torch.cuda.stream(side):
        step(spare, *held)
    torch.cuda.current_stream().wait_stream(side)
    del spare
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(model, *held)
    for k in range(4):
        data = types.roll(k), desc.roll(k, 0) * (1 + k), target
        for a, b in zip(held, data):
            a.copy_(b)
        graph.replay()
        want = step(twin, *data)
        torch.cuda.synchronize()
        assert norm > 0.01 and torch.equal(norm, want)
        assert all(torch.equal(p, q) for p, q in zip(model.parameters(), twin.parameters()))


def test_example_runs():
    found = node_blocks.fit(steps=3, cells=2, channels=32, blocks=1, report=None, by_species=True, clip=1.0, form="integers")
    assert all(math.isfinite(v) for v in found.values())
