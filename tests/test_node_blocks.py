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


# ---- masked atoms ----


def _with_masked(n=30):
    """Atoms with masked ones among them, whose descriptors are anything; which ones are real."""
    types, desc = _inputs(n)
    types[3], types[10], types[11], types[29] = -1, 5, 1 << 40, -(1 << 40)
    there = (types >= 0) & (types < 5)
    desc[3], desc[10, 2], desc[11] = float("nan"), float("inf"), 1e30
    return types, desc, there


def test_masked_atoms_have_no_energy_and_teach_nothing():
    model = _head()
    torch.nn.init.normal_(model.shift)
    types, desc, there = _with_masked()
    desc.requires_grad_()
    w = torch.randn(30)
    e = model(types, desc)
    assert (e[~there] == 0).all()
    (e * w).sum().backward()
    got = {k: v.grad.clone() for k, v in model.named_parameters()}
    slopes = desc.grad.clone()
    assert (slopes[~there] == 0).all()
    model.zero_grad()
    desc2 = desc.detach()[there].requires_grad_()
    e2 = model(types[there], desc2)
    (e2 * w[there]).sum().backward()
    # the same sums over the atoms with zeros among them: FP32 roundings
    torch.testing.assert_close(e[there], e2, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(slopes[there], desc2.grad, rtol=1e-5, atol=1e-6)
    for k, v in model.named_parameters():
        torch.testing.assert_close(got[k], v.grad, rtol=1e-5, atol=1e-5, msg=k)


@pytest.mark.parametrize("blocks", [0, 2])
def test_masked_atoms_served(blocks):
    model = node_blocks.NodeBlocks(5, 12, 16, blocks)
    torch.nn.init.normal_(model.shift)
    types, desc, there = _with_masked()
    e = model.serve()(types, desc)
    assert (e[~there] == 0).all()
    torch.testing.assert_close(e[there], model.serve()(types[there], desc[there]), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(e, model(types, desc), rtol=1e-5, atol=1e-6)


# ---- types ----


def test_weights_of_a_16_bit_head_get_gradients_of_their_own_type():
    model = _head(dtype=torch.bfloat16)
    types, desc = _inputs()
    model(types, desc).square().sum().backward()
    for w in (model.lift, *model.weights):
        # of FP32 sums, of which bf16 holds one in 2^16
        assert w.grad.dtype is torch.float32
        assert (w.grad.bfloat16().float() == w.grad).float().mean() < 0.1


@pytest.mark.parametrize("name", ["embed", "norm", "residual", "linear"])
def test_gradients_of_a_graph_are_changed_in_place(name):
    """As any gradient may be whose own derivatives nobody asks for."""
    call, leaf = _calls()[name]
    y = call()
    want, = torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
    got, = torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)
    got.mul_(2.0)
    assert torch.equal(got, 2 * want)
