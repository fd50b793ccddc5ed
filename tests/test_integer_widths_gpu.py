"""GPU tests of rows brought to 8-bit integers at the largest widths that are accepted."""

import pytest
import torch

from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [(1 << 31) - 2049, (1 << 31) - 2041, (1 << 31) - 513])
def test_widest_rows(cols):
    """Columns up to 2^31 - 513, where a step past the row's end is past 2^31: values of every part of the row's last step."""
    x = torch.zeros(1, cols, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, cols // 2, cols - 2500, cols - 2048, cols - 1030, cols - 515, cols - 9, cols - 8, cols - 2, cols - 1])
    x[0, at] = torch.tensor([127.0, 1, -2, 3, -4, 5, -6, 7, -8, 9, -10], dtype=torch.bfloat16, device="cuda")
    b = ops.quantize_integers(x)
    assert b.scales.item() == 1.0 and b.values.shape == (1, -(-cols // 128) * 128)
    assert b.values[0, at].tolist() == [127, 1, -2, 3, -4, 5, -6, 7, -8, 9, -10]
    assert torch.count_nonzero(b.values).item() == len(at)
