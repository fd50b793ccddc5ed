"""GPU test of the head with masked atoms (types outside its table): zero energies, nothing learned from them, and the
others as without them."""

import math

import pytest
import torch

from symmetrix import node_blocks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_atoms(index, dtype):
    torch.manual_seed(6)
    model = node_blocks.NodeBlocks(5, 24, 64, 2, dtype).cuda()
    torch.nn.init.normal_(model.shift)
    n, more = 100, 20  # the masked atoms are the last, so that the others share their 8-bit blocks with zeros alone
    types = torch.randint(0, 5, (n + more,), device="cuda", dtype=index)
    types[n:] = torch.tensor([-1, 5, torch.iinfo(index).max, torch.iinfo(index).min], device="cuda").repeat(5).to(index)
    desc, w = torch.randn(n + more, 24, device="cuda"), torch.randn(n + more, device="cuda")
    desc[n + 1], desc[n + 2, 3], desc[n + 3] = math.nan, math.inf, 1e30
    e = model(types, desc)
    assert (e[n:] == 0).all()
    (e * w).sum().backward()
    got = {k: v.grad.clone() for k, v in model.named_parameters()}
    model.zero_grad()
    e2 = model(types[:n], desc[:n])
    (e2 * w[:n]).sum().backward()
    # rows on their own; the readout's sum of 64 terms by a library, in FP32
    torch.testing.assert_close(e[:n], e2, rtol=1e-5, atol=1e-6)
    for k, v in model.named_parameters():
        # sums over the atoms, in FP32 and another order
        assert (got[k] - v.grad).norm() <= 2.0 ** -18 * v.grad.norm() + 1e-12, k
    served = model.serve()
    torch.testing.assert_close(served(types, desc)[:n], served(types[:n], desc[:n]), rtol=1e-5, atol=1e-6)
    assert (served(types, desc)[n:] == 0).all()
