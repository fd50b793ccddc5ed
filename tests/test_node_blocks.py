"""CPU tests of the head's autograd functions and of what lies around its operators (symmetrix.node_blocks), over plain
operators."""

import pytest
import torch

import _node_plain
from symmetrix import node_blocks


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    monkeypatch.setattr(node_blocks, "ops", _node_plain)
    torch.manual_seed(11)


def _head(**more):
    return node_blocks.NodeBlocks(5, 12, 16, 2, **more)


def _inputs(n=30):
    return torch.randint(0, 5, (n,)), torch.randn(n, 12)


# ---- second derivatives ----


def _calls():
    x, both = torch.randn(6, 8, requires_grad=True), torch.randn(6, 16, requires_grad=True)
    w, v = torch.randn(8, 8, requires_grad=True), torch.rand(8, requires_grad=True)
    types = torch.tensor([0, 1, 1, 3, -1, 7])
    return {"embed": (lambda: node_blocks._Embed.apply(w, types, 2.0), w),
            "norm": (lambda: node_blocks._Norm.apply(x, v, 1e-6), x),
            "residual": (lambda: sum(node_blocks._GatedResidual.apply(x, both, v, v, v, 1e-6)), both),
            "linear": (lambda: node_blocks._Linear.apply(x, w), x)}


@pytest.mark.parametrize("name", ["embed", "norm", "residual", "linear"])
@pytest.mark.parametrize("seed_needs_grad", [False, True])
def test_second_derivatives_raise(name, seed_needs_grad):
    call, leaf = _calls()[name]
    y = call()
    seed = torch.randn(y.shape, requires_grad=seed_needs_grad)
    want, = torch.autograd.grad(y, leaf, seed, retain_graph=True)
    assert not want.requires_grad
    got, = torch.autograd.grad(y, leaf, seed, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        got.square().sum().backward()


@pytest.mark.parametrize("frozen", [False, True])
def test_loss_of_forces_raises(frozen):
    """Energies and their slopes in one loss: the slopes' part is refused, also where the readout asks for no gradient."""
    model = _head()
    model.readout.requires_grad_(not frozen)
    types, desc = _inputs()
    desc.requires_grad_()
    slope, = torch.autograd.grad(model(types, desc).sum(), desc, create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        slope.square().sum().backward()


def test_slopes_alone_are_formed():
    model = _head()
    types, desc = _inputs()
    desc.requires_grad_()
    slope, = torch.autograd.grad(model(types, desc).sum(), desc)
    way, h = torch.randn_like(desc), 1e-3
    with torch.no_grad():
        change = (model(types, desc + h * way) - model(types, desc - h * way)).sum() / (2 * h)
    # O(h^2) of the third derivative, and FP32 roundings of 30 energies of size 1 (2^-20) over 2h
    assert abs(change - (slope * way).sum()) < 5e-3 * (1 + abs(change))
