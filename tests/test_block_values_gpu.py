"""GPU tests of products with copied and saved 8-bit weights, and of weights loaded from the CPU's copy."""

import copy
import io

import pytest
import torch

from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 7, 90])
def test_products_with_copies(m):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(m, 333, generator=g, device="cuda")
    w = ops.quantize(torch.randn(70, 333, generator=g, device="cuda"))
    want = ops.block_linear(x, w)
    f = io.BytesIO()
    torch.save(w, f)
    copies = [copy.deepcopy(w)]
    w.values.view(torch.uint8).zero_()  # the original's bytes are another matrix's now
    w.scales.zero_()
    for where in ("cuda", "cpu"):
        f.seek(0)
        w2 = torch.load(f, map_location=where)
        copies.append(ops.BlockValues(w2.values.cuda(), w2.scales.cuda(), w2.shape))
    for c in copies:
        assert torch.equal(ops.block_linear(x, c), want)
        assert torch.equal(ops.block_product(ops.quantize(x), c), ops.block_linear(x, c, torch.float32))
