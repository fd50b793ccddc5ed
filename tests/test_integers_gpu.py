"""GPU tests of the products in 8-bit integers against their definition: integers and scales exactly, products to
the roundings that the definition names."""

import copy
import math

import pytest
import torch

from _node_reference import assert_within, d
from symmetrix import node_ops as ops
from symmetrix._native import lib

pytestmark = pytest.mark.gpu

UNIT_127 = float.fromhex("0x1.020408p-7")  # the FP32 number next to 1/127
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(17)


def _rows(gen, r, c, dtype):
    x = torch.randn(r, c, generator=gen, device="cuda") * torch.exp(torch.randn(r, 1, generator=gen, device="cuda"))
    return x.to(dtype)


def _by_hand(x):
    """(integers, FP32 scales) of finite x, in float64 on the CPU."""
    x = d(x)
    top = x.abs().amax(1) if x.shape[1] else torch.zeros(len(x)).double()
    scale = (top * UNIT_127).float().clamp(min=2.0 ** -126)  # (a product of two FP32 numbers is exact in float64)
    return torch.round(x / scale.double()[:, None]), scale


def _view(t, offset, more):
    r, c = t.shape
    wide = torch.full((r * (c + more) + offset,), math.nan, dtype=t.dtype, device=t.device)
    v = wide[offset:].view(r, c + more)[:, :c]
    v.copy_(t)
    return v


SHAPES = [(0, 5), (1, 1), (3, 7), (5, 0), (17, 127), (16, 128), (33, 129), (100, 511), (9, 512), (64, 1000), (7, 1024), (5, 2041),
          (300, 2048), (3, 4095), (2, 8192), (3, 8193), (2, 20001), (20000, 40)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r, c", SHAPES)
def test_quantize(gen, r, c, dtype):
    x = _rows(gen, r, c, dtype)
    for given in (x, _view(x, 1, 3)):
        b = ops.quantize_integers(given)
        q, scale = _by_hand(x)
        assert b.shape == (r, c) and torch.equal(b.scales.cpu(), scale)
        assert torch.equal(b.values[:, :c].cpu().double(), q) and not b.values[:, c:].any()
        assert torch.equal(d(b.float()), (q.float() * scale[:, None]).double())


def test_ties_zeros_and_small_rows():
    x = torch.zeros(6, 40, device="cuda")
    x[1] = torch.arange(40) / 2 - 10
    x[1, 0], x[2, 3], x[3, 5] = 127.0, 2.0 ** -149, 3.4e38
    x[4] = 2.0 ** -120 * (torch.arange(40) - 20.0)
    x[5] = torch.linspace(-1, 1, 40)
    b = ops.quantize_integers(x)
    q, scale = _by_hand(x)
    assert scale[0] == 2.0 ** -126 and scale[1] == 1 and scale[2] == 2.0 ** -126
    assert torch.equal(b.scales.cpu(), scale) and torch.equal(b.values[:, :40].cpu().double(), q)
    assert b.values[1, 1:6].tolist() == [-10, -9, -8, -8, -8] and b.values[3, 5] == 127


def test_quotients_next_to_ties(gen):
    """x at (q + 1/2) scale, and the values beside it: the quotient's own rounding may not move them over the border."""
    top = 1 + torch.rand(200, generator=gen, device="cuda")
    scale = (top.double() * UNIT_127).float()
    tie = (torch.arange(126, device="cuda").double() + 0.5)[None] * scale.double()[:, None]
    tie = tie.float()
    up, down = torch.nextafter(tie, tie + 1), torch.nextafter(tie, tie - 1)
    x = torch.cat([top[:, None], tie, up, down, -tie, -up, -down], 1)
    b = ops.quantize_integers(x)
    q, s = _by_hand(x)
    assert torch.equal(b.scales.cpu(), s) and torch.equal(b.values[:, :x.shape[1]].cpu().double(), q)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_rows_that_are_no_numbers(gen, bad):
    for m in (5, 40):
        x, w = _rows(gen, m, 200, F32), ops.quantize_integers(_rows(gen, 30, 200, F32))
        fine = ops.integer_linear(x, w)
        x[3, 199] = bad
        b = ops.quantize_integers(x)
        assert torch.isnan(b.scales[3]) and not b.values[3].any() and torch.isfinite(b.scales[[0, 1, 2, 4]]).all()
        y = ops.integer_linear(x, w)
        assert torch.isnan(y[3]).all()
        others = torch.arange(m) != 3
        assert torch.equal(y[others], fine[others])


PRODUCTS = [(0, 4, 8), (4, 0, 8), (3, 5, 0), (1, 1, 1), (1, 40, 1000), (2, 17, 129), (16, 33, 500), (17, 31, 64), (40, 70, 4096),
            (65, 64, 128), (200, 130, 257), (129, 1000, 224), (1, 8200, 384), (600, 300, 1300), (1030, 2050, 128),
            (4096, 4100, 256), (2100, 4200, 384), (7, 50, 131072), (33, 40, 131072)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m, n, k", PRODUCTS)
def test_products(gen, m, n, k, dtype):
    x, w = _rows(gen, m, k, dtype), _rows(gen, n, k, dtype)
    a, b = ops.quantize_integers(x), ops.quantize_integers(w)
    qa, qb = a.values[:, :k].double(), b.values[:, :k].double()
    # (sums of whole numbers below 2^53: exact on the card in float64, whatever their order)
    want = (torch.matmul(qa, qb.T.contiguous()) * (a.scales.double()[:, None] * b.scales.double()[None])).cpu()
    for out in (F32, dtype):
        got = ops.integer_product(a, b, out)
        assert got.dtype is out and got.shape == (m, n)
        assert_within(got, want, 3.0001 * 2.0 ** -24 * want.abs())
        assert torch.equal(ops.integer_linear(x, b, out), got)
    assert torch.equal(ops.integer_linear(x, b), ops.integer_product(a, b, dtype))


@pytest.mark.parametrize("m", [3, 100])
def test_longest_sums_are_exact(m):
    """2^17 products of 127 by 127, the largest sum: 2,114,060,288 is a whole number of FP32."""
    k = 1 << 17
    x, w = torch.full((m, k), 127.0, device="cuda"), torch.full((20, k), -127.0, device="cuda")
    got = ops.integer_linear(x, ops.quantize_integers(w))
    assert (got == -float(k * 127 * 127)).all()


@pytest.mark.parametrize("m", [3, 100])
def test_integers_of_another_making(m):
    """Values down to -128, which rows brought to integers do not reach: the largest sum is 2^31."""
    k = 1 << 17
    a, b = (ops.IntegerValues(torch.full((rows, k), -128, dtype=torch.int8, device="cuda"), torch.ones(rows, device="cuda"), (rows, k))
            for rows in (m, 20))
    assert (ops.integer_product(a, b) == 2.0 ** 31).all()
    b.values[:] = 127
    assert (ops.integer_product(a, b) == -float(k * 128 * 127)).all()


def test_finer_than_blocks(gen):
    """What the form is for: rows of normal values, a quarter of the 8-bit blocks' error."""
    x, w = torch.randn(512, 1024, generator=gen, device="cuda"), torch.randn(256, 1024, generator=gen, device="cuda")
    want = d(x) @ d(w).T
    off = [(d(y) - want).norm().item() for y in (ops.integer_linear(x, ops.quantize_integers(w)),
                                                 ops.block_linear(x, ops.quantize(w)))]
    # uniform steps of max/127, about 3.5/127 of a normal row's deviation, round by 0.29 of that: 0.8% for each operand;
    # a 4-bit significand rounds by 2.6%
    assert off[0] < 0.5 * off[1]


def test_views_streams_and_graphs(gen):
    w = ops.quantize_integers(_rows(gen, 96, 300, BF16))
    for m in (3, 70):
        data = [_rows(gen, m, 300, BF16) for _ in range(3)]
        held = _view(data[0], 3, 5)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.integer_linear(held, w)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.integer_linear(held, w)
        for x in data:
            with torch.cuda.stream(side):
                want = ops.integer_linear(x, w)
            held.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_copies(gen, tmp_path):
    b = ops.quantize_integers(_rows(gen, 30, 200, F16))
    torch.save(b, tmp_path / "w.pt")
    for c in (copy.deepcopy(b), torch.load(tmp_path / "w.pt"), ops.IntegerValues(b.values.clone(), b.scales.clone(), b.shape)):
        assert c.shape == b.shape and torch.equal(c.values, b.values) and torch.equal(c.scales, b.scales)
        assert c.values.data_ptr() != b.values.data_ptr()


def test_rows_behind_the_outputs_stay(gen):
    for m in (9, 300):
        x, w = _rows(gen, m, 200, BF16), ops.quantize_integers(_rows(gen, 50, 200, BF16))
        want = ops.integer_linear(x, w)
        out = torch.full((m + 3, 57), 5.0, dtype=BF16, device="cuda")
        size = lib.smx_integer_linear_workspace(m, 50, 200)
        room = torch.full((size + 64,), 77, dtype=torch.uint8, device="cuda")
        assert lib.smx_integer_linear(x.data_ptr(), 200, 1, w.values.data_ptr(), w.scales.data_ptr(), m, 50, 200, 1, out.data_ptr(), 57,
                                      room.data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out[:m, :50], want) and (out[m:] == 5).all() and (out[:, 50:] == 5).all() and (room[size:] == 77).all()


def test_offsets_beyond_32_bits(gen):
    """x in rows that lie 2^22 values apart."""
    far = torch.empty(1100 << 22, dtype=BF16, device="cuda")
    x = far.view(1100, 1 << 22)[:, :200]
    x.copy_(_rows(gen, 1100, 200, BF16))
    w = ops.quantize_integers(_rows(gen, 50, 200, BF16))
    assert torch.equal(ops.integer_linear(x, w), ops.integer_linear(x.contiguous(), w))
