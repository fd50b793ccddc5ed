"""GPU tests of rows by type: the plan, the products with a matrix for each type and their gradients, against
their definitions in float64: no rows, one, many; odd widths, strides and alignments; masked rows and types
without rows; infinities and NaN beside what a sum takes; offsets beyond 32 bits; streams and graphs."""

import math

import pytest
import torch

from _node_reference import assert_within, d
from symmetrix import node_ops as ops
from symmetrix._native import lib

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(11)


def _normal(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _types(gen, rows, v, kind, dtype=torch.int32):
    if kind == "one":
        z = torch.full((rows,), v - 1, device="cuda")
    elif kind == "none":
        z = torch.full((rows,), -1, device="cuda")
    elif kind == "few":  # of many types three, very unequal
        z = torch.tensor([0, v // 2, v - 1], device="cuda")[
            (torch.rand(rows, generator=gen, device="cuda") ** 3 * 3).long().clamp(0, 2)]
    else:
        z = torch.randint(0, v, (rows,), generator=gen, device="cuda")
        if kind == "outside":
            z[::3] = -1
            z[1::7] = v
            z[2::11] = (1 << 40) + 1 if dtype is torch.int64 else (1 << 31) - 1
    return z.to(dtype)


def _view(t, offset, more, fill=math.nan):
    """t's values in a view of wider rows that starts `offset` values in, the rest `fill`."""
    lead, c = t.shape[:-1], t.shape[-1]
    rows = math.prod(lead)
    wide = torch.full((rows * (c + more) + offset,), fill, dtype=t.dtype, device=t.device)
    v = wide[offset:].view(rows, c + more)[:, :c]
    v.copy_(t.reshape(rows, c))
    return v.unflatten(0, lead) if len(lead) > 1 else v


def _by_hand(z, v):
    z = z.cpu().long()
    z = torch.where((z >= 0) & (z < v), z, v)
    order = torch.sort(z, stable=True).indices
    return z, order, torch.searchsorted(z[order], torch.arange(v + 1))


# ---- the plan ----

PLAN = [(0, 5, "any"), (1, 1, "any"), (1, 89, "none"), (63, 2, "any"), (64, 255, "outside"), (65, 256, "outside"),
        (135, 89, "few"), (2047, 3, "outside"), (2048, 4096, "any"), (2049, 1, "one"), (2049, 4096, "outside"),
        (4097, 255, "any"), (5000, 89, "few"), (5001, 1023, "any"), (5001, 1024, "any"), (20000, 10, "any"),
        (70001, 1009, "outside"), (131071, 2, "few"), (300000, 4096, "any"), (300001, 7, "none"), (1100000, 300, "any")]


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("rows, v, kind", PLAN)
def test_group_rows(gen, rows, v, kind, index):
    z = _types(gen, rows, v, kind, index)
    groups = ops.group_rows(z, v)
    _, order, offsets = _by_hand(z, v)
    assert groups.order.dtype is torch.int32 and groups.offsets.dtype is torch.int32
    assert torch.equal(groups.order.cpu().long(), order)
    assert torch.equal(groups.offsets.cpu().long(), offsets)


# ---- the products ----

# rows, types, inputs, outputs: kinds of few rows (their own kernel), tiles of 64, 128 and 256, runs of rows that are cut
CASES = [(0, 3, 8, 8, "any"), (1, 1, 1, 1, "any"), (1, 64, 40, 24, "any"), (1, 5, 2048, 72, "any"), (5, 3, 0, 8, "any"),
         (7, 3, 8, 0, "any"), (16, 1, 64, 64, "any"), (17, 1, 64, 64, "any"), (33, 7, 100, 36, "outside"),
         (64, 89, 33, 17, "any"), (147, 32, 128, 96, "any"), (200, 4, 65, 1, "outside"), (135, 89, 32, 64, "few"),
         (300, 3, 24, 999, "none"), (513, 2, 224, 99, "one"), (700, 1, 8, 16, "any"), (1025, 3, 31, 200, "few"),
         (1500, 89, 224, 120, "outside"), (2048, 2, 64, 1024, "any"), (2500, 5, 72, 1032, "few"),
         (3001, 2, 130, 260, "any"), (4100, 1, 72, 4104, "any"), (5000, 10, 64, 136, "any"), (6791, 89, 56, 80, "any")]


def _grouped_by_hand(z, v, x, w, grad):
    """(y, dx, dw) and the sums of their terms' magnitudes, in float64 on the CPU."""
    z, _, _ = _by_hand(z, v)
    x, w, grad = d(x), d(w), d(grad)
    y, dx, dw = torch.zeros(len(z), w.shape[1]).double(), torch.zeros(x.shape).double(), torch.zeros(w.shape).double()
    sizes = [torch.zeros_like(t) for t in (y, dx, dw)]
    for g in torch.unique(z).tolist():
        if g == v:
            continue
        at = z == g
        y[at], dx[at], dw[g] = x[at] @ w[g].T, grad[at] @ w[g], grad[at].T @ x[at]
        xa, wa, ga = x[at].abs(), w[g].abs(), grad[at].abs()
        sizes[0][at], sizes[1][at], sizes[2][g] = xa @ wa.T, ga @ wa, ga.T @ xa
    return (y, dx, dw), sizes


def _check(z, v, x, w, grad, dtype=None):
    """All three against float64.  A sum of FP32 rounds each of its terms once, by 2^-24 of a partial sum that the
    magnitudes bound; FP32 products leave out 2^-24 of each term and round six parts."""
    groups = ops.group_rows(z, v)
    want, sizes = _grouped_by_hand(z, v, x, w, grad)
    got = [ops.grouped_linear(x, w, groups, dtype), *ops.grouped_linear_gradient(grad, x, w, groups)]
    counts = torch.bincount(_by_hand(z, v)[0], minlength=v + 1)
    terms = [x.shape[1], w.shape[1], int(counts[:v].max()) if len(z) else 0]
    assert [t.dtype for t in got] == [dtype or x.dtype, x.dtype, F32]
    for t, a, s, k in zip(got, want, sizes, terms):
        # (products of FP32 values below 2^-110 lose up to 2^-134 each: nothing at these sizes)
        assert_within(t, a, (k + 8 + (16 if x.dtype is F32 else 0)) * 2.0 ** -23 * s)
    return groups, got


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows, v, k, n, kind", CASES)
def test_grouped_linear_both_ways(gen, rows, v, k, n, kind, dtype):
    z = _types(gen, rows, v, kind)
    x, w, grad = _normal(gen, rows, k, dtype=dtype), _normal(gen, v, n, k, dtype=dtype), _normal(gen, rows, n, dtype=dtype)
    _check(z, v, x, w, grad)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows, v, k, n, kind", [(40, 30, 64, 96, "any"), (90, 3, 136, 264, "outside"), (700, 2, 40, 100, "few"),
                                                 (1200, 1, 129, 33, "any")])
def test_views_beside_nan(gen, rows, v, k, n, kind, dtype):
    """Rows that start anywhere and lie apart, NaN between them: nothing of it is taken in."""
    z = _types(gen, rows, v, kind)
    x, w, grad = _normal(gen, rows, k, dtype=dtype), _normal(gen, v, n, k, dtype=dtype), _normal(gen, rows, n, dtype=dtype)
    for offset, more in ((0, 8), (8, 16), (1, 3), (3, 0)):
        _check(z, v, _view(x, offset, more), _view(w, offset, more), _view(grad, offset, more))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS[1:])
def test_outputs_in_float32(gen, dtype):
    for rows, v in ((30, 20), (600, 2)):
        z = _types(gen, rows, v, "outside")
        x, w, grad = _normal(gen, rows, 70, dtype=dtype), _normal(gen, v, 50, 70, dtype=dtype), _normal(gen, rows, 50, dtype=dtype)
        _check(z, v, x, w, grad, F32)
        groups = ops.group_rows(z, v)
        wide = ops.grouped_linear_gradient(grad, x, w, groups)[1]
        assert torch.equal(ops.grouped_linear_gradient(grad, x, w, groups, dtype)[1], wide.to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows, v, k, n", [(30, 20, 72, 40), (900, 3, 72, 136), (1400, 2, 33, 50)])
def test_infinities_stay_where_they_belong(gen, rows, v, k, n, dtype):
    """Infinite and NaN values in masked rows, in a type without rows and in one row: rows and types without them
    have the results that they have alone."""
    z = _types(gen, rows, v, "any")
    z[z == 1] = 0
    z[5], z[8] = -1, v + 3
    x, w, grad = _normal(gen, rows, k, dtype=dtype), _normal(gen, v, n, k, dtype=dtype), _normal(gen, rows, n, dtype=dtype)
    groups, plain = _check(z, v, x, w, grad)
    x[5], grad[5], x[8, 0], grad[8, n - 1] = math.nan, math.inf, -math.inf, math.nan
    w[1, 0] = math.nan
    w[1, n - 1] = math.inf
    got = [ops.grouped_linear(x, w, groups), *ops.grouped_linear_gradient(grad, x, w, groups)]
    for a, b in zip(plain, got):
        assert torch.equal(a, b)
    # one row of its type: its own outputs, and its type's weights' gradient
    x[0, 3], grad[0, 2] = math.inf, math.nan
    y, (dx, dw) = ops.grouped_linear(x, w, groups), ops.grouped_linear_gradient(grad, x, w, groups)
    assert not torch.isfinite(y[0]).any() and torch.equal(y[1:], plain[0][1:])
    assert torch.isnan(dx[0]).all() and torch.equal(dx[1:], plain[1][1:])
    others = torch.arange(v, device="cuda") != z[0]
    assert torch.equal(dw[others], plain[2][others])
    mine = dw[z[0].item()]
    assert torch.isnan(mine[2]).all() and not torch.isfinite(mine[:, 3]).any()
    rest = torch.ones_like(mine, dtype=torch.bool)
    rest[2] = False
    rest[:, 3] = False
    assert torch.equal(mine[rest], plain[2][z[0].item()][rest])


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_gradients_against_differences(gen, dtype):
    """The product is linear in both inputs, so its differences are its derivatives: <g, f(x + u, w) - f(x, w)> is
    <dx, u>, and so for w.  (Values are small whole numbers, whose sums are exact in every type.)"""
    rows, v, k, n = 700, 4, 40, 24
    z = _types(gen, rows, v, "outside")

    def whole(*shape):
        return torch.randint(-2, 3, shape, generator=gen, device="cuda").to(dtype)
    x, u, w, m, grad = whole(rows, k), whole(rows, k), whole(v, n, k), whole(v, n, k), whole(rows, n)
    groups = ops.group_rows(z, v)

    def f(x, w):
        return ops.grouped_linear(x, w, groups, F32).double()
    dx, dw = ops.grouped_linear_gradient(grad, x, w, groups)
    assert (grad.double() * (f(x + u, w) - f(x, w))).sum() == (dx.double() * u.double()).sum()
    assert (grad.double() * (f(x, w + m) - f(x, w))).sum() == (dw.double() * m.double()).sum()


def test_same_bits_again(gen):
    z = _types(gen, 5000, 3, "few")
    x, w, grad = _normal(gen, 5000, 64), _normal(gen, 3, 48, 64), _normal(gen, 5000, 48)
    groups = ops.group_rows(z, 3)
    first = [ops.grouped_linear(x, w, groups), *ops.grouped_linear_gradient(grad, x, w, groups)]
    for _ in range(3):
        again = [ops.grouped_linear(x, w, groups), *ops.grouped_linear_gradient(grad, x, w, groups)]
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_one_gradient_alone(gen):
    z = _types(gen, 300, 3, "any")
    x, w, grad = _normal(gen, 300, 40, dtype=BF16), _normal(gen, 3, 24, 40, dtype=BF16), _normal(gen, 300, 24, dtype=BF16)
    groups = ops.group_rows(z, 3)
    dx, dw = ops.grouped_linear_gradient(grad, x, w, groups)
    a, none = ops.grouped_linear_gradient(grad, None, w, groups)
    assert none is None and torch.equal(a, dx)
    none, b = ops.grouped_linear_gradient(grad, x, None, groups)
    assert none is None and torch.equal(b, dw)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_rows_beyond_32_bits(gen, dtype):
    """Rows whose offsets pass 2^32 values, and a matrix that does."""
    rows, v, k, n, stride = 1100, 2, 32, 40, 1 << 22
    z = _types(gen, rows, v, "any")
    x, w, grad = _normal(gen, rows, k, dtype=dtype), _normal(gen, v, n, k, dtype=dtype), _normal(gen, rows, n, dtype=dtype)
    far = torch.empty(rows * stride, dtype=dtype, device="cuda")
    wide = far.view(rows, stride)[:, :k]
    wide.copy_(x)
    _check(z, v, wide, w, grad)
    apart = far[:2 * ((rows // 2) * stride)].view(2, -1)[:, :n * k].view(2, n, k)
    apart.copy_(w)
    _check(z, v, x, apart, grad)
    del far


def test_rows_behind_the_outputs_stay(gen):
    """At the C boundary, outputs in wider rows: what lies between and behind them is not written."""
    for rows, v, k, n in ((20, 9, 40, 24), (700, 2, 40, 24), (700, 2, 33, 23)):
        z = _types(gen, rows, v, "outside")
        x, w, grad = _normal(gen, rows, k, dtype=BF16), _normal(gen, v, n, k, dtype=BF16), _normal(gen, rows, n, dtype=BF16)
        groups = ops.group_rows(z, v)
        want = [ops.grouped_linear(x, w, groups), *ops.grouped_linear_gradient(grad, x, w, groups)]
        s = torch.cuda.current_stream().cuda_stream
        y, dx = torch.full((rows + 2, n + 5), 7.0, dtype=BF16, device="cuda"), torch.full((rows + 2, k + 3), 7.0, dtype=BF16, device="cuda")
        dw = torch.full((v + 1, n + 1, k + 9), 7.0, device="cuda")
        plan = groups._room.data_ptr()
        assert lib.smx_grouped_linear(x.data_ptr(), k, 1, w.data_ptr(), k, n * k, plan, rows, v, k, n, 1, y.data_ptr(), n + 5, s) == 0
        assert lib.smx_grouped_linear_by_rows(grad.data_ptr(), n, 1, w.data_ptr(), k, n * k, plan, rows, v, k, n, 1,
                                              dx.data_ptr(), k + 3, s) == 0
        size = lib.smx_grouped_linear_by_weights_workspace(rows, v, k, n)
        room = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
        assert lib.smx_grouped_linear_by_weights(grad.data_ptr(), n, x.data_ptr(), k, 1, plan, rows, v, k, n, 0, dw.data_ptr(),
                                                 k + 9, (n + 1) * (k + 9), room.data_ptr(), size, s) == 0
        for got, a in ((y, want[0]), (dx, want[1])):
            assert torch.equal(got[:rows, :a.shape[1]], a)
            assert (got[rows:] == 7).all() and (got[:, a.shape[1]:] == 7).all()
        assert torch.equal(dw[:v, :n, :k], want[2])
        assert (dw[v:] == 7).all() and (dw[:, n:] == 7).all() and (dw[:, :, k:] == 7).all()


def test_streams_and_graphs(gen):
    """A captured step (plan, product, both gradients) replayed with new inputs, between eager steps on another stream."""
    rows, v, k, n = 3000, 5, 48, 64
    zs = [_types(gen, rows, v, kind) for kind in ("any", "outside", "few", "none", "one")]
    data = [(_normal(gen, rows, k, dtype=BF16), _normal(gen, v, n, k, dtype=BF16), _normal(gen, rows, n, dtype=BF16))
            for _ in zs]

    def step(z, x, w, grad):
        groups = ops.group_rows(z, v)
        return [ops.grouped_linear(x, w, groups), *ops.grouped_linear_gradient(grad, x, w, groups)]
    held = [zs[0].clone(), *(t.clone() for t in data[0])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for z, parts in zip(zs, data):
        with torch.cuda.stream(side):
            other = step(z, *parts)
        for a, b in zip(held, (z, *parts)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, other))
