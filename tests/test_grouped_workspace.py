"""CPU tests of the weights' gradient's workspace: none where a type's tiles fill the card by themselves, so that no type is cut,
and room for every run where types may be."""

import pytest

from symmetrix._native import lib

size = lib.smx_grouped_linear_by_weights_workspace


@pytest.mark.parametrize("rows, v, k, n", [(8192, 1, 8192, 8192), (2048, 1, 16384, 16384), (100000, 89, 16384, 8192),
                                           (1 << 20, 1, 1 << 14, 1 << 14)])
def test_nothing_to_cut(rows, v, k, n):
    assert size(rows, v, k, n) == 0


@pytest.mark.parametrize("rows, v, k, n", [(30000, 2, 256, 512), (20000, 10, 512, 1024), (6791, 89, 224, 999), (5000, 3, 8, 6)])
def test_types_may_be_cut(rows, v, k, n):
    """A type of all the rows in runs of 512 or more: two parts for each at most, of a matrix each."""
    got = size(rows, v, k, n)
    assert got >= 4 * 2 * 2 * k * n and got % (4 * k * n) == 0 and got <= 4 * 2 * (rows // 512 + 1) * k * n
