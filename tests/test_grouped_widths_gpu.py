"""GPU tests of the products by type at sizes that pass one launch of the kernel of few rows."""

import pytest
import torch

from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu


def test_most_outputs_of_few_rows():
    """A row or so of each of 4,096 types through more outputs than a launch has threads for (4,352 units of 64 columns with 128
    threads each pass 2^32 from 493,000 columns on)."""
    v, rows, n = 4096, 4096, (1 << 19) + 3
    gen = torch.Generator(device="cuda").manual_seed(37)
    z = torch.randint(-1, v, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    x = torch.randn(rows, 1, generator=gen, device="cuda").to(torch.bfloat16)
    w = torch.empty(v, n, 1, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    y = ops.grouped_linear(x, w, ops.group_rows(z, v))
    # (one term: rounded once, as torch's product is)
    want = torch.where((z >= 0)[:, None], x * w[z.clamp(min=0).long(), :, 0], 0)
    assert torch.equal(y, want)
