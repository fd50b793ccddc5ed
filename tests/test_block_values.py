"""CPU tests of BlockValues (symmetrix.node_ops): what its bytes stand for however they are given, and copies."""

import copy
import io
import pickle

import pytest
import torch

from symmetrix import node_ops

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _bytes(r=3, c=200):
    """Values and scales of a matrix [r][c] as uint8, and the matrix."""
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-8, 9, (r, 256), generator=g).float()
    x[:, c:] = 0
    scales = torch.zeros(r, 4, dtype=torch.uint8)
    scales[:, :2] = torch.randint(120, 130, (r, 2), generator=g)
    size = torch.exp2(scales[:, :2].float() - 127).repeat_interleave(128, 1)
    return x.to(E4M3).view(torch.uint8), scales, (x * size)[:, :c]


@pytest.mark.parametrize("value_type", [torch.uint8, E4M3])
@pytest.mark.parametrize("scale_type", [torch.uint8, E8M0])
def test_bytes_are_e4m3_and_e8m0(value_type, scale_type):
    values, scales, want = _bytes()
    b = node_ops.BlockValues(values.view(value_type), scales.view(scale_type), want.shape)
    assert b.values.dtype is E4M3 and b.scales.dtype is torch.uint8
    assert torch.equal(b.float(), want)
    assert b.values.data_ptr() == values.data_ptr() and b.scales.data_ptr() == scales.data_ptr()


@pytest.mark.parametrize("kind", [torch.int8, torch.bool, torch.float8_e5m2, torch.float8_e4m3fnuz])
def test_other_bytes_are_refused(kind):
    values, scales, want = _bytes()
    with pytest.raises(ValueError, match="values must be contiguous bytes"):
        node_ops.BlockValues(values.view(kind), scales, want.shape)
    with pytest.raises(ValueError, match="scales must be contiguous bytes"):
        node_ops.BlockValues(values, scales.view(kind), want.shape)


def _saved(b):
    f = io.BytesIO()
    torch.save({"weights": [b]}, f)
    f.seek(0)
    return torch.load(f)["weights"][0]


COPIES = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda b: pickle.loads(pickle.dumps(b)), "save": _saved}


@pytest.mark.parametrize("way", list(COPIES))
@pytest.mark.parametrize("together", [False, True])
def test_copies_have_their_own_addresses(way, together):
    values, scales, want = _bytes()
    if together:  # as the operators make them: one allocation
        b = node_ops.BlockValues._empty(*want.shape, want)
        b.values.copy_(values.view(E4M3))
        b.scales.copy_(scales)
    else:
        b = node_ops.BlockValues(values, scales, want.shape)
    c = COPIES[way](b)
    assert type(c) is node_ops.BlockValues and c.shape == b.shape
    assert c._at == (c.values.data_ptr(), c.scales.data_ptr())
    assert torch.equal(c.float(), want)
    if way == "copy":  # shares the tensors, as torch's own do
        assert c._at == b._at
        return
    room = [range(t.data_ptr(), t.data_ptr() + t.numel()) for t in (b.values, b.scales)]
    assert not any(at in r for at in c._at for r in room)
    b.values.view(torch.uint8).zero_()
    assert torch.equal(c.float(), want)


def test_addresses_are_those_of_the_call():
    """Memory that was put in another place under the same tensor is read where it is."""
    values, scales, want = _bytes()
    b = node_ops.BlockValues(values, scales, want.shape)
    other = b.values.clone()
    b.values.set_(other)
    assert b._at[0] == other.data_ptr()
