"""CPU tests of BlockValues (symmetrix.node_ops): what its bytes stand for however they are given."""

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
