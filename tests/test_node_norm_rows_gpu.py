"""GPU tests of the residual norm's gradient where each workgroup works on several rows: the rows read ahead, the places
in LDS used again from row to row, and the sums over a workgroup's rows."""

import pytest
import torch

from test_node_ops_gpu import BF16, F16, F32, _check_norm, gen  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("r, c, gate, dtype", [
    (4500, 520, "full", BF16), (6791, 999, "channel", F32), (4501, 1024, "row", F16), (2100, 1027, "row", F32),
    (2101, 2048, "full", BF16), (1100, 2100, "none", F32), (1101, 4100, "row", BF16), (1100, 4096, "full", F32),
    (900, 5000, "full", F16), (700, 10001, "channel", BF16)],
    ids=lambda v: str(v).replace("torch.", ""))
def test_many_rows_of_a_workgroup(gen, r, c, gate, dtype):  # noqa: F811
    _check_norm(gen, r, c, gate, dtype)


@pytest.mark.parametrize("r, c", [(4500, 600), (1100, 4096)])
def test_same_bits_every_time(gen, r, c):  # noqa: F811
    from symmetrix import node_ops as ops
    x, dd, gate, gy, gh = (torch.randn(r, c, generator=gen, device="cuda") for _ in range(5))
    w = torch.ones(c, device="cuda")
    want = ops.residual_norm_gradient(x, dd, w, gate, w, w, gy, gh)
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(ops.residual_norm_gradient(x, dd, w, gate, w, w, gy, gh), want))
