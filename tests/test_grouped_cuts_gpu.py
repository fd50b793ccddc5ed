"""GPU tests of the products by type at sizes that reach each of their kernels' cuts: 64 and 16 columns of few rows and their
waves, tiles of 256, 128 and 64, more types than a wave has lanes, kinds of one row and of many, runs that are cut and not."""

import pytest
import torch

from symmetrix import node_ops as ops
from test_grouped_gpu import BF16, F16, F32, _check, _normal, _types, gen  # noqa: F401 (gen: a fixture)

pytestmark = pytest.mark.gpu

FEW = [(600, 300, 40, 1100, "any"), (600, 300, 1100, 1100, "outside"), (40, 40, 4160, 840, "any"), (600, 300, 39, 1101, "any"),
       (30, 20, 4160, 72, "any"), (300, 20, 64, 2049, "few"), (3, 700, 2000, 700, "any"), (1, 1, 8, 20000, "any")]
TILES = [(4096, 1, 72, 4104, "any"), (3000, 3, 264, 3080, "few"), (6000, 70, 64, 520, "any"), (9000, 100, 40, 1040, "outside"),
         (5000, 300, 72, 136, "few"), (20000, 2, 40, 72, "any"), (20000, 90, 40, 72, "few"), (33000, 1, 16, 24, "one"),
         (2600, 5, 520, 1032, "any"), (2600, 5, 519, 1033, "few"), (17000, 1000, 24, 32, "any")]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, v, k, n, kind", FEW + TILES)
def test_every_cut(gen, rows, v, k, n, kind, dtype):  # noqa: F811
    z = _types(gen, rows, v, kind)
    x, w, grad = _normal(gen, rows, k, dtype=dtype), _normal(gen, v, n, k, dtype=dtype), _normal(gen, rows, n, dtype=dtype)
    torch.full((rows, n), float("nan"), dtype=dtype, device="cuda")  # (so that what is not written is seen)
    _check(z, v, x, w, grad)


@pytest.mark.parametrize("rows, v, n", [(600, 300, 1100), (300, 20, 2049), (5000, 80, 136)])
def test_masked_rows_are_zeros_everywhere(gen, rows, v, n):  # noqa: F811
    z = torch.full((rows,), -1, device="cuda", dtype=torch.int32)
    z[rows // 2] = v - 1
    x, w = _normal(gen, rows, 40, dtype=BF16), _normal(gen, v, n, 40, dtype=BF16)
    torch.full((rows, n), float("nan"), dtype=BF16, device="cuda")
    y = ops.grouped_linear(x, w, ops.group_rows(z, v))
    others = torch.arange(rows, device="cuda") != rows // 2
    assert not y[others].any() and y[rows // 2].abs().sum() > 0
