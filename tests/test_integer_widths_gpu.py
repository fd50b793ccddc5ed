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


@pytest.mark.parametrize("m", [2, 9])
def test_most_columns_of_few_rows(m):
    """More columns than one launch has threads for (2^27 columns of 32 threads each are 2^32)."""
    n, k, slice_ = (1 << 27) + 21, 40, 1 << 26
    w = ops.IntegerValues(torch.zeros(n, 128, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda"), (n, k))
    at = torch.tensor([0, 1, slice_ - 1, slice_, slice_ + 17, 2 * slice_ - 1, 2 * slice_, 2 * slice_ + 16, n - 2, n - 1])
    w.values[at, :k] = torch.arange(1, 11, dtype=torch.int8, device="cuda")[:, None]
    w.scales[at[3:]] = 0.5
    x = torch.ones(m, k, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 127.0  # (scale 1)
    want = (127 + k - 1) * torch.arange(1.0, 11.0) * torch.tensor([1.0] * 3 + [0.5] * 7)
    for y in (ops.integer_linear(x, w, torch.float32), ops.integer_product(ops.quantize_integers(x), w)):
        assert torch.equal(y[:, at].cpu(), want.expand(m, 10)) and torch.count_nonzero(y).item() == 10 * m
        del y
