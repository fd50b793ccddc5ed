"""CPU tests of the head with weights by species and of its served forms (symmetrix.node_blocks), over plain operators."""

import types as _module

import pytest
import torch

import _node_plain
from symmetrix import node_blocks


def group_rows(types, num_types):
    return torch.where((types >= 0) & (types < num_types), types, num_types).long()


def grouped_linear(x, w, groups, dtype=None):
    y = x.new_zeros(x.shape[0], w.shape[1])
    for g in range(w.shape[0]):
        y[groups == g] = x[groups == g] @ w[g].T
    return y


def grouped_linear_gradient(grad, x, w, groups, dtype=None):
    dx = None if w is None else grad.new_zeros(grad.shape[0], w.shape[2])
    n = int(groups.max()) + 1
    dw = None if x is None else torch.zeros(5, grad.shape[1], x.shape[1], dtype=dtype or torch.float32)
    for g in range(min(n, 5)):
        at = groups == g
        if w is not None:
            dx[at] = grad[at] @ w[g]
        if x is not None:
            dw[g] = (grad[at].float().T @ x[at].float()).to(dw.dtype)
    return dx, dw


def quantize_integers(x):
    return x.clone()


def integer_linear(x, w, dtype=None):
    return _node_plain.block_linear(x, w, dtype)


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    ops = _module.SimpleNamespace(**{k: v for k, v in vars(_node_plain).items() if not k.startswith("_")})
    for f in (group_rows, grouped_linear, grouped_linear_gradient, quantize_integers, integer_linear):
        setattr(ops, f.__name__, f)
    monkeypatch.setattr(node_blocks, "ops", ops)
    torch.manual_seed(23)


def _head(**more):
    return node_blocks.NodeBlocks(5, 12, 16, 2, by_species=True, **more)


def test_species_share_nothing():
    """The weights of a species get gradients from its atoms alone, and change no other's energy."""
    model = _head()
    assert model.weights[0].shape == (5, 32, 16)
    types, desc = torch.tensor([0, 1, 1, 3, -1, 7, 0]), torch.randn(7, 12)
    e = model(types, desc)
    assert (e[4:6] == 0).all()
    e[types == 1].sum().backward()
    for w in model.weights:
        assert w.grad[1].abs().sum() > 0 and not w.grad[[0, 2, 3, 4]].any()
    with torch.no_grad():
        model.weights[0][1] += 1
        assert torch.equal(model(types, desc)[types != 1], e[types != 1])
        assert not torch.equal(model(types, desc)[types == 1], e[types == 1])


def test_one_species_is_the_shared_head():
    a, b = _head(), node_blocks.NodeBlocks(5, 12, 16, 2)
    with torch.no_grad():
        for p, q in zip(a.parameters(), b.parameters()):
            q.copy_(p[3] if p.dim() == 3 else p)
    types, desc = torch.full((9,), 3), torch.randn(9, 12)
    torch.testing.assert_close(a(types, desc), b(types, desc))


def test_gradients_against_differences():
    """The species' linear is linear in both inputs, so its differences are its derivatives; small whole numbers are exact."""
    def whole(*shape):
        return torch.randint(-3, 4, shape).float()
    groups = group_rows(torch.tensor([0, 1, 1, 4, 2, 0, -1]), 5)
    x, w, grad = whole(7, 8).requires_grad_(), whole(5, 4, 8).requires_grad_(), whole(7, 4)
    u, m = whole(7, 8), whole(5, 4, 8)
    f = node_blocks._SpeciesLinear.apply
    y = f(x, w, groups)
    y.backward(grad)
    assert (grad * (f(x + u, w, groups) - y)).sum() == (x.grad * u).sum()
    assert (grad * (f(x, w + m, groups) - y)).sum() == (w.grad * m).sum()


@pytest.mark.parametrize("by_species", [False, True])
@pytest.mark.parametrize("form", ["blocks", "integers"])
def test_served_forms(form, by_species):
    model = node_blocks.NodeBlocks(5, 12, 16, 2, by_species=by_species)
    types, desc = torch.randint(-1, 6, (30,)), torch.randn(30, 12)
    torch.testing.assert_close(model.serve(form)(types, desc), model(types, desc).detach())


def test_refusals():
    with pytest.raises(ValueError, match="blocks or integers"):
        _head().serve("bits")
    model = _head()
    desc = torch.randn(6, 12, requires_grad=True)
    slope, = torch.autograd.grad(model(torch.tensor([0, 1, 1, 4, 2, 0]), desc).sum(), desc, create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        slope.square().sum().backward()


def test_weights_of_another_type():
    x, w = torch.randn(6, 8, dtype=torch.bfloat16, requires_grad=True), torch.randn(5, 4, 8, requires_grad=True)
    groups = group_rows(torch.tensor([0, 1, 1, 4, 2, 0]), 5)
    y = node_blocks._SpeciesLinear.apply(x, w, groups)
    y.sum().backward()
    assert y.dtype is x.grad.dtype is torch.bfloat16 and w.grad.dtype is torch.float32
    v = w.detach().to(torch.bfloat16).requires_grad_()
    node_blocks._SpeciesLinear.apply(x, v, groups).sum().backward()
    assert v.grad.dtype is torch.bfloat16
