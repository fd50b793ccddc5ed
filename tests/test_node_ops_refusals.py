"""CPU tests of refusals by the node operators' Python functions that come before any allocation or launch: on CPU
tensors a function that got as far as its launch would complain of the device instead."""

import pytest
import torch

from symmetrix import node_ops


def _blocks(r, c):
    pitch = -(-c // 128) * 128
    return node_ops.BlockValues(torch.zeros(r, pitch, dtype=torch.uint8), torch.zeros(r, -(-pitch // 512) * 4, dtype=torch.uint8),
                                (r, c))


def test_embed_gradient():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="int32 or int64 vector"):
        node_ops.embed_gradient(torch.tensor(3), x, 5)
    with pytest.raises(ValueError, match="int32 or int64 vector"):
        node_ops.embed_gradient(torch.zeros(4, 1, dtype=torch.int64), x, 5)
    with pytest.raises(ValueError, match="num_types"):
        node_ops.embed_gradient(torch.zeros(4, dtype=torch.int64), x, -1)


def test_linear_and_its_gradient():
    x, grad = torch.zeros(4, 8), torch.zeros(4, 6)
    w, w_columns, x_columns = _blocks(6, 8), _blocks(8, 6), _blocks(8, 4)
    with pytest.raises(ValueError, match="products are"):
        node_ops.block_linear(x, w, torch.float64, keep=True)
    with pytest.raises(ValueError, match="products are"):
        node_ops.block_linear_gradient(grad, w_columns, x_columns, torch.int32)
    with pytest.raises(ValueError, match="w_columns must have as many columns"):
        node_ops.block_linear_gradient(grad, w, x_columns)
    with pytest.raises(ValueError, match="x_columns must have as many columns"):
        node_ops.block_linear_gradient(grad, w_columns, w)
    with pytest.raises(ValueError, match="x_columns must be BlockValues"):
        node_ops.block_linear_gradient(grad, w_columns, x)
    with pytest.raises(ValueError, match="two-dimensional"):
        node_ops.block_linear_gradient(grad[0], w_columns, x_columns)
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.block_linear_gradient(grad, w_columns, x_columns)
