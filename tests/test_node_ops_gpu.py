"""GPU tests of the node operators against their definitions in float64 (tests/_node_reference.py): sizes
from nothing to many rows, odd widths, strides and alignments, masked types, zero and non-finite
rows, offsets beyond 32 bits, streams, graphs, and gradients against differences."""

import math

import pytest
import torch

from _node_reference import LEAST, UNIT, Norm, assert_within, d, product, quantized
from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(7)


def _normal(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _view(t, offset, more):
    """t's values in a view of wider rows that starts `offset` values in."""
    r, c = t.shape
    wide = torch.empty(r * (c + more) + offset, dtype=t.dtype, device=t.device)
    v = wide[offset:].view(r, c + more)[:, :c] if r else wide[:0].view(0, c)
    v.copy_(t)
    return v


# ---- species embedding ----


def _types(gen, tokens, v, kind, dtype):
    if kind == "one":
        z = torch.full((tokens,), v - 1, device="cuda")
    elif kind == "none":
        z = torch.full((tokens,), -1, device="cuda")
    else:
        z = torch.randint(0, v, (tokens,), generator=gen, device="cuda")
        if kind == "outside":  # below, just past and far past the table
            z[::3] = -1
            z[1::7] = v
            z[2::11] = (1 << 40) + 1 if dtype is torch.int64 else (1 << 31) - 1
    return z.to(dtype)


EMBED = [(0, 5, 8, "any"), (1, 1, 1, "any"), (1, 89, 128, "any"), (63, 2, 3, "any"), (65, 7, 100, "outside"),
         (300, 89, 32, "none"), (1000, 3, 257, "one"), (1000, 256, 64, "any"), (1000, 257, 33, "outside"),
         (5000, 89, 128, "outside"), (5001, 2, 96, "any"), (4097, 70001, 40, "outside"), (40000, 300, 24, "any"),
         (9000, 66000, 16, "any"), (30, 40, 2050, "any"), (256, 5, 600, "any"), (257, 5, 600, "any"),
         (255, 20000, 96, "outside"), (200, 2, 20, "any"), (1024, 1024, 70, "outside"), (1025, 3, 40, "any"),
         (900, 1025, 48, "outside"), (257, 1, 700, "any"), (600, 1, 1, "any"), (700, 4, 2041, "outside"),
         (2000, 3, 9, "outside"), (3001, 4, 2048, "any"), (2500, 2, 511, "outside"), (20011, 1, 130, "any"),
         (30000, 4, 65, "outside"), (90001, 3, 31, "any"), (1500, 4, 2049, "any"), (700, 4, 300, "none")]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("tokens, v, c, kind", EMBED)
def test_embed_both_ways(gen, tokens, v, c, kind, index, dtype):
    z = _types(gen, tokens, v, kind, index)
    table, grad = _normal(gen, v, c, dtype=dtype), _normal(gen, tokens, c, dtype=dtype)
    scale = math.sqrt(c)
    s64 = torch.tensor(scale, dtype=F32).double().item()
    zc = z.cpu().long()
    good = (zc >= 0) & (zc < v)
    want = torch.zeros(tokens, c, dtype=torch.float64)
    want[good] = d(table)[zc[good]] * s64
    # one product in FP32, rounded, then rounded to the type
    assert_within(ops.embed(z, table, scale), want, 2.0 ** -24 * want.abs())
    got = ops.embed_gradient(z, grad, v, scale)
    total, size = torch.zeros(v, c, dtype=torch.float64), torch.zeros(v, c, dtype=torch.float64)
    total.index_add_(0, zc[good], d(grad)[good])
    size.index_add_(0, zc[good], d(grad)[good].abs())
    count = torch.zeros(v, dtype=torch.float64).index_add_(0, zc[good], torch.ones(int(good.sum()), dtype=torch.float64))
    assert_within(got, total * s64, (count + 2)[:, None] * 2.0 ** -24 * size * s64)
    assert torch.equal(got, ops.embed_gradient(z, grad, v, scale))  # the same bits again


@pytest.mark.parametrize("dtype, c, more", [(F32, 1023, 1), (BF16, 2050, 0), (F16, 2048, 8)], ids=IDS)
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
def test_embed_of_many_rows(gen, dtype, c, more, index):
    """Outputs of over 200 MB, against the same rows in parts of a fiftieth."""
    z = _types(gen, 51_203, 301, "outside", index)
    table = _normal(gen, 301, c, dtype=dtype)
    out = ops.embed(z, _view(table, 0, more), 1.7)
    for i in range(0, z.numel(), 1000):
        assert torch.equal(out[i:i + 1000], ops.embed(z[i:i + 1000].contiguous(), table, 1.7)), i


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("offset, more", [(0, 8), (1, 0), (3, 5)])
def test_embed_strides(gen, offset, more, dtype):
    z = _types(gen, 500, 11, "any", torch.int64)
    table, grad = _normal(gen, 11, 40, dtype=dtype), _normal(gen, 500, 40, dtype=dtype)
    assert torch.equal(ops.embed(z, _view(table, offset, more), 0.5), ops.embed(z, table, 0.5))
    assert torch.equal(ops.embed_gradient(z, _view(grad, offset, more), 11), ops.embed_gradient(z, grad, 11))


def test_embed_gradient_of_differences(gen):
    """<gradient, direction> against the change of the loss along it (linear: any step will do)."""
    z = _types(gen, 200, 9, "outside", torch.int32)
    table, way, w = _normal(gen, 9, 24), _normal(gen, 9, 24), _normal(gen, 200, 24)

    def loss(t):
        return (d(ops.embed(z, t, 0.7)) * d(w)).sum().item()
    slope = (d(ops.embed_gradient(z, w, 9, 0.7)) * d(way)).sum().item()
    # 4,800 terms of size 1 rounded to 2^-24 each, and the gradient's own rounding
    assert abs((loss(table + way) - loss(table - way)) / 2 - slope) < 4800 * 2.0 ** -22


def test_embed_infinities_stay_in_their_rows(gen):
    z = torch.tensor([0, 1, 2, 1, 0, -1], device="cuda")
    grad = _normal(gen, 6, 16)
    grad[1, 3], grad[5, 2] = math.inf, math.nan  # the second in a masked row
    out = ops.embed_gradient(z, grad, 3)
    assert out[1, 3] == math.inf
    out[1, 3] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("c", [3, 41, 200, 700])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_embed_gradient_of_few_species(gen, dtype, c):
    """Views of any alignment, and infinities that stay with their type and out of the masked rows."""
    z = _types(gen, 3000, 3, "outside", torch.int64)
    z[1], z[2] = 1, -1
    grad = _normal(gen, 3000, c, dtype=dtype)
    want = ops.embed_gradient(z, grad, 3)
    for offset, more in ((0, 8), (1, 0), (3, 5)):
        assert torch.equal(ops.embed_gradient(z, _view(grad, offset, more), 3), want)
    grad[1, c - 1], grad[2, 0] = math.inf, math.nan
    out = ops.embed_gradient(z, grad, 3)
    assert out[1, c - 1] == math.inf
    out[1, c - 1] = want[1, c - 1]
    assert torch.equal(out, want)


# ---- residual norm ----


def _norm_inputs(gen, r, c, gate, dtype, full=True):
    x, dd = _normal(gen, r, c, dtype=dtype), 3 * _normal(gen, r, c, dtype=dtype)
    g = {"none": None, "full": (r, c), "channel": (c,), "row": (r, 1)}[gate]
    g = 2 * _normal(gen, *g, dtype=dtype) if g else None
    post, scale, nxt = (1 + 0.3 * _normal(gen, c) for _ in range(3))
    if not full:
        scale, nxt = None, None
    return x, dd, post, g, scale, nxt


NORM = [(0, 8), (1, 1), (1, 4096), (2, 2), (3, 31), (70, 64), (5, 100), (130, 128), (4, 129), (9, 256), (33, 300),
        (40, 512), (7, 999), (12, 1024), (3, 2050), (6, 2048), (2, 4100), (3, 8192), (2, 10001), (2, 16384)]


def _check_norm(gen, r, c, gate, dtype, full=True, eps=1e-6, view=lambda t: t):
    x, dd, post, g, scale, nxt = _norm_inputs(gen, r, c, gate, dtype, full)
    if gate == "full" and r:
        both = torch.cat([dd, g], 1)
        dd, g = both[:, :c], both[:, c:]
    f = Norm(x, dd, post, g, scale, nxt, eps)
    x, dd = view(x), view(dd)
    y, h = ops.residual_norm(x, dd, post, g, scale, nxt, eps=eps)
    assert_within(y, f.y, f.y_bound)
    if nxt is None:
        assert h is None
    else:
        assert_within(h, f.h, f.h_bound)
    gy, gh = _normal(gen, r, c, dtype=dtype), _normal(gen, r, c, dtype=dtype) if full else None
    got = ops.residual_norm_gradient(x, dd, post, g, scale, nxt, view(gy), gh, eps=eps)
    want, bound = f.backward(gy, gh)
    for name, t, given in zip(("x", "d", "gate", "post", "scale", "next"), got, (x, dd, g, post, scale, nxt)):
        assert (t is None) == (given is None), name
        if t is not None:
            assert_within(t, want[name], bound[name])
    again = ops.residual_norm_gradient(x, dd, post, g, scale, nxt, view(gy), gh, eps=eps)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r, c", NORM)
def test_norm_sizes(gen, r, c, dtype):
    _check_norm(gen, r, c, "full" if c > 1 else "channel", dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("gate", ["none", "channel", "row"])
@pytest.mark.parametrize("r, c", [(1, 1), (37, 64), (300, 129), (2500, 128), (5, 3001), (11, 4096)])
def test_norm_gates(gen, r, c, gate, dtype):
    if gate == "row" and c == 1:
        gate = "channel"
    _check_norm(gen, r, c, gate, dtype)


@pytest.mark.parametrize("gate", ["none", "full", "row"])
@pytest.mark.parametrize("r, c", [(3, 33), (65, 256), (2, 5000)])
def test_norm_without_scale_and_next(gen, r, c, gate):
    _check_norm(gen, r, c, gate, BF16, full=False)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("offset, more", [(0, 8), (0, 1), (1, 0), (3, 5)])
@pytest.mark.parametrize("c", [64, 96, 1000])
def test_norm_strides(gen, c, offset, more, dtype):
    _check_norm(gen, 17, c, "row", dtype, view=lambda t: _view(t, offset, more))


def test_norm_many_rows(gen):
    _check_norm(gen, 20001, 96, "channel", F32)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r, c", [(1, 1), (1, 4096), (33, 100), (5, 129), (70, 128), (3, 1000), (2, 16384), (9, 2048)])
def test_plain_norm(gen, r, c, dtype):
    x, w = _normal(gen, r, c, dtype=dtype), 1 + 0.3 * _normal(gen, c)
    f = Norm(x, None, None, None, None, w, 1e-6)
    assert_within(ops.norm(x, w), f.h, f.h_bound)
    gh = _normal(gen, r, c, dtype=dtype)
    got = ops.residual_norm_gradient(x, None, None, None, None, w, None, gh)
    want, bound = f.backward(None, gh)
    assert_within(got[0], want["x"], bound["x"])
    assert_within(got[5], want["next"], bound["next"])
    assert got[1:5] == (None,) * 4
    q = ops.norm(x, w, quantized=True)
    _check_near_blocks(q, f.h, f.h_bound)


def _check_near_blocks(q, want, bound):
    """Blocks of a value that is itself off by `bound`: the scale is the one of a magnitude in its
    range, and each value is within that range and half a step of E4M3 (2^-4 of it, or 2^-10 of the scale)."""
    r, c = want.shape
    blocks = -(-c // 128)
    pad = torch.zeros(r, blocks * 128 - c, dtype=torch.float64)
    mag = torch.cat([want.abs(), pad], 1).view(r, blocks, 128)
    off = torch.cat([bound.expand_as(want), pad], 1).view(r, blocks, 128)
    byte = q.scales.cpu()[:, :blocks].long()
    low = quantized((mag - off).clamp(min=0).view(r, -1))[1]
    high = quantized((mag + off).view(r, -1))[1]
    assert ((byte >= low) & (byte <= high)).all()
    assert (q.scales.cpu()[:, blocks:] == 0).all()
    step = torch.exp2(byte.double() - 127 - 10)[:, :, None].expand(r, blocks, 128).reshape(r, -1)[:, :c]
    got = d(q.float())
    assert ((got - want).abs() <= bound + torch.maximum(step, (want.abs() + bound) * 2.0 ** -4)).all()
    assert (q.values.view(torch.uint8)[:, c:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r, c", [(1, 4096), (70, 100), (9, 512), (3, 5001)])
def test_residual_norm_in_blocks(gen, r, c, dtype):
    x, dd, post, g, scale, nxt = _norm_inputs(gen, r, c, "channel", dtype)
    f = Norm(x, dd, post, g, scale, nxt, 1e-6)
    y, h = ops.residual_norm(x, dd, post, g, scale, nxt, quantized=True)
    assert_within(y, f.y, f.y_bound)
    _check_near_blocks(h, f.h, f.h_bound)


@pytest.mark.parametrize("gate", ["none", "full", "channel", "row"])
def test_norm_gradient_against_differences(gen, gate):
    r, c = 5, 40
    names = ("x", "d", "post", "gate", "scale", "next")
    v = dict(zip(names, _norm_inputs(gen, r, c, gate, F32)))
    gy, gh = _normal(gen, r, c), _normal(gen, r, c)

    def loss(v):
        y, h = ops.residual_norm(v["x"], v["d"], v["post"], v["gate"], v["scale"], v["next"])
        return (d(y) * d(gy) + d(h) * d(gh)).sum().item()
    got = dict(zip(("x", "d", "gate", "post", "scale", "next"),
                   ops.residual_norm_gradient(*(v[n] for n in names), gy, gh)))
    for n in names:
        if v[n] is None:
            continue
        way = _normal(gen, *v[n].shape)

        def slope(h):
            return (loss({**v, n: v[n] + h * way}) - loss({**v, n: v[n] - h * way})) / (2 * h)
        # Richardson: h^4 of the fifth derivative (h = 1/32: about 1e-6), and 400 values of about 1 that are off by 2^-22,
        # over 2h
        h = 1 / 32
        near = (4 * slope(h / 2) - slope(h)) / 3
        want = (d(got[n]) * d(way)).sum().item()
        assert abs(near - want) < 2e-3 * (1 + abs(want)), n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("c", [96, 2048])
def test_norm_rows_of_zeros_and_non_finite_rows(gen, c, dtype):
    x, dd, post, g, scale, nxt = _norm_inputs(gen, 6, c, "full", dtype)
    x[0], dd[0] = 0, 0       # 1 / sqrt(eps) times nothing
    x[1, 3] = math.inf       # y and its norm: the row's h is not a number or zero, y keeps its infinity
    dd[2, 5] = math.nan
    g[3, :] = -math.inf      # a closed gate
    g[4, :] = math.inf       # an open one
    y, h = ops.residual_norm(x, dd, post, g, scale, nxt)
    assert (y[0] == 0).all() and (h[0] == 0).all()
    assert y[1, 3] == math.inf and torch.isfinite(y[1, 4:]).all() and torch.isnan(h[1, 3]) and (h[1, 4:] == 0).all()
    assert torch.isnan(y[2]).all() and torch.isnan(h[2]).all()
    assert torch.equal(y[3], x[3])
    f = Norm(x[4:], dd[4:], post, torch.cat([torch.full_like(g[4:5], 60000), g[5:]]), scale, nxt, 1e-6)
    f.rel = (c + 64) * 2.0 ** -22
    assert_within(y[4:], f.y, f.rel * (f.y - f.x).abs() + 2.0 ** -22 * f.y.abs())
    gy, gh = _normal(gen, 6, c, dtype=dtype), _normal(gen, 6, c, dtype=dtype)
    dx, d_d, dg, *_ = ops.residual_norm_gradient(x, dd, post, g, scale, nxt, gy, gh)
    for r in (3, 4, 5):
        assert torch.isfinite(dx[r]).all() and torch.isfinite(d_d[r]).all() and torch.isfinite(dg[r]).all()
    assert (dg[3] == 0).all() and (dg[4] == 0).all() and (d_d[3] == 0).all()


def test_norm_outputs_in_place_of_inputs(gen):
    from symmetrix import _native
    import ctypes
    x, dd, post, g, scale, nxt = _norm_inputs(gen, 50, 200, "row", BF16)
    y, _ = ops.residual_norm(x, dd, post, g, scale)
    a = _native.SmxResidualNormArgs(*ops._norm_inputs(x, dd, post, g, scale, None, 1e-6), x.data_ptr(), 200)
    _native.check(_native.lib.smx_residual_norm(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(x, y)


# ---- 8-bit blocks ----


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("r, c", [(1, 1), (3, 128), (128, 3), (130, 129), (5, 600), (257, 100), (300, 1030)])
def test_quantize_both_ways(gen, r, c, dtype):
    x = _normal(gen, r, c, dtype=dtype) * torch.exp(_normal(gen, r, c)).to(dtype)
    x[:, ::3] *= 0.001
    x[0] = 0
    rows, cols = ops.quantize(x, columns=True)
    for got, src in ((rows, x), (cols, x.T)):
        want, byte = quantized(src)
        assert got.shape == tuple(src.shape)
        assert torch.equal(d(got.float()), want)
        blocks = byte.shape[1]
        assert torch.equal(got.scales.cpu()[:, :blocks].long(), byte)
        assert (got.scales[:, blocks:] == 0).all()
        assert (got.values.view(torch.uint8)[:, src.shape[1]:] == 0).all()
    one, other = ops.quantize(x), ops.quantize(x, rows=False, columns=True)
    assert torch.equal(one.values.view(torch.uint8), rows.values.view(torch.uint8)) and torch.equal(one.scales, rows.scales)
    assert torch.equal(other.values.view(torch.uint8), cols.values.view(torch.uint8)) and torch.equal(other.scales, cols.scales)


def test_quantize_extremes():
    x = torch.zeros(5, 256, device="cuda")
    x[0, 0], x[0, 1], x[0, 128] = 3.4e38, 1.0, 2.0 ** -140
    x[1, :4] = torch.tensor([448.0, 447.9, 1.0625, 2.0 ** -10])
    x[2, 0], x[2, 1], x[2, 2], x[2, 130] = math.inf, -math.inf, math.nan, 5.0
    x[3, 0], x[3, 1] = 2.0 ** -149, 2.0 ** -126
    x[4] = -0.0
    rows, cols = ops.quantize(x, columns=True)
    for got, src in ((rows, x), (cols, x.T)):
        want, byte = quantized(src)
        assert torch.equal(torch.isnan(want), torch.isnan(d(got.float())))
        assert torch.equal(got.scales.cpu()[:, :byte.shape[1]].long(), byte)
        # (the decoded value of a scale of 2^-127 is a subnormal product: compare the 8-bit values)
        scale = torch.exp2((byte - 127).double()).repeat_interleave(128, 1)[:, :src.shape[1]]
        assert torch.equal(torch.nan_to_num(d(got.values.float())[:, :src.shape[1]] * scale), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("offset, more", [(0, 8), (1, 0), (3, 5)])
def test_quantize_strides(gen, offset, more, dtype):
    x = _normal(gen, 70, 200, dtype=dtype)
    for a, b in zip(ops.quantize(_view(x, offset, more), columns=True), ops.quantize(x, columns=True)):
        assert torch.equal(a.values.view(torch.uint8), b.values.view(torch.uint8)) and torch.equal(a.scales, b.scales)


LINEAR = [(0, 8, 8), (1, 1, 1), (1, 16, 128), (1, 1000, 513), (2, 64, 300), (7, 33, 4096), (15, 128, 128),
          (16, 255, 129), (17, 16, 1000), (31, 512, 2048), (33, 100, 64), (64, 64, 64), (65, 4097, 130), (100, 1, 100),
          (128, 128, 512), (129, 300, 260), (200, 1030, 1), (257, 512, 640), (300, 257, 2050), (513, 300, 127),
          (1000, 520, 1024), (30, 5000, 700), (520, 20, 9000), (70, 1001, 5000), (700, 1300, 1500)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m, n, k", LINEAR)
def test_linear_sizes(gen, m, n, k, dtype):
    x, w = _normal(gen, m, k, dtype=dtype), _normal(gen, n, k, dtype=dtype) / math.sqrt(k)
    wq = ops.quantize(w)
    a, b = quantized(x)[0], quantized(w)[0]
    want, bound = product(a, b)
    y = ops.block_linear(x, wq)
    assert y.dtype is dtype
    assert_within(y, want, bound)
    y32, xt = ops.block_linear(x, wq, dtype=F32, keep=True)
    assert_within(y32, want, bound)
    if m:
        assert torch.equal(d(xt.float()), quantized(x.T)[0])


# products of more tiles than the card holds at once, and of each tile's size, with edges in both directions
MANY_TILES = [(2500, 2501, 200), (2500, 2499, 300), (4090, 4085, 140), (4090, 4085, 300), (4100, 4098, 260),
              (8190, 4091, 130), (8190, 4091, 260), (100_000, 60, 130), (100_001, 61, 390)]


@pytest.mark.parametrize("m, n, k", MANY_TILES)
def test_product_of_many_tiles(gen, m, n, k):
    x, w = ops.quantize(_normal(gen, m, k, dtype=BF16)), ops.quantize(_normal(gen, n, k) / math.sqrt(k))
    a, b = d(x.float()), d(w.float())
    want, bound = product(a, b)
    for dtype in TYPES:
        assert_within(ops.block_product(x, w, dtype), want, bound)


def test_linear_without_inputs(gen):
    w = ops.quantize(torch.empty(5, 0, device="cuda"))
    assert torch.equal(ops.block_linear(torch.empty(3, 0, device="cuda"), w), torch.zeros(3, 5, device="cuda"))


@pytest.mark.parametrize("m, n, k", [(1, 70, 300), (40, 200, 300), (300, 600, 300)])
def test_linear_non_finite(gen, m, n, k):
    x, w = _normal(gen, m, k), _normal(gen, n, k)
    x[m // 2, 7] = math.inf
    w[3, k - 1] = math.nan
    y = ops.block_linear(x, ops.quantize(w))
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[m // 2], bad[:, 3] = True, True
    assert torch.equal(torch.isnan(y), bad)


@pytest.mark.parametrize("m, n, k", [(3, 50, 300), (64, 130, 200), (300, 200, 600)])
def test_linear_far_scales(gen, m, n, k):
    """Rows and blocks of very different size: scales from far apart meet in one sum."""
    x = _normal(gen, m, k) * torch.exp2(torch.randint(-60, 60, (m, 1), generator=gen, device="cuda").float())
    w = _normal(gen, n, k) * torch.exp2(torch.randint(-60, 60, (n, 1), generator=gen, device="cuda").float())
    w[:, 128:] *= 2.0 ** 12
    a, b = quantized(x)[0], quantized(w)[0]
    want, bound = product(a, b)
    # (some meet beyond FP32: partial sums of those outputs may be infinities of both signs)
    beyond = a.abs() @ b.abs().T > torch.finfo(F32).max
    assert beyond.double().mean() < 0.2
    y = ops.block_linear(x, ops.quantize(w))
    assert_within(torch.where(beyond.cuda(), 0.0, y), torch.where(beyond, 0.0, want), bound)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m, n, k", [(1, 8, 8), (40, 130, 70), (300, 257, 512), (1000, 96, 200)])
def test_linear_gradient(gen, m, n, k, dtype):
    x, w, g = (_normal(gen, *s, dtype=dtype) for s in ((m, k), (n, k), (m, n)))
    w_rows, w_cols = ops.quantize(w, columns=True)
    _, xt = ops.block_linear(x, w_rows, keep=True)
    dx, dw = ops.block_linear_gradient(g, w_cols, xt)
    assert dx.dtype is dtype and dw.dtype is F32
    assert_within(dx, *product(quantized(g)[0], quantized(w.T)[0]))
    assert_within(dw, *product(quantized(g.T)[0], quantized(x.T)[0]))
    # and of the unrounded product: two operands that are off by 2^-4 of a value, or 2^-10 of the largest of its block
    exact, size = d(g) @ d(w), d(g).abs() @ d(w).abs()
    top = 2.0 ** -9 * d(g).abs().amax(1, keepdim=True) @ d(w).abs().sum(0, keepdim=True)
    top = top + 2.0 ** -9 * d(g).abs().sum(1, keepdim=True) @ d(w).abs().amax(0, keepdim=True)
    assert ((d(dx) - exact).abs() <= (2.0 ** -3 + 2.0 ** -7) * size + top).all()


def test_linear_gradient_against_differences(gen):
    """On values that 8 bits hold exactly (small whole numbers) the gradient is that of the loss."""
    def whole(*s):
        return torch.randint(-4, 5, s, generator=gen, device="cuda").float()
    x, w, g = whole(20, 40), whole(30, 40), whole(20, 30)
    w_rows, w_cols = ops.quantize(w, columns=True)
    _, xt = ops.block_linear(x, w_rows, keep=True)
    dx, dw = ops.block_linear_gradient(g, w_cols, xt)

    def loss(x, w):
        return (d(ops.block_linear(x, ops.quantize(w))) * d(g)).sum().item()
    ways = whole(20, 40), whole(30, 40)
    assert loss(x + ways[0], w) - loss(x - ways[0], w) == 2 * (d(dx) * d(ways[0])).sum().item()
    assert loss(x, w + ways[1]) - loss(x, w - ways[1]) == 2 * (d(dw) * d(ways[1])).sum().item()


def test_product_of_strided_views(gen):
    x, w = _normal(gen, 90, 333, dtype=BF16), ops.quantize(_normal(gen, 70, 333))
    for offset, more in ((0, 8), (1, 0), (3, 4)):
        for m in (1, 5, 90):
            assert torch.equal(ops.block_linear(_view(x[:m], offset, more), w), ops.block_linear(x[:m], w))


# ---- all of them ----


def _calls(gen):
    """One call of each operator, as functions of nothing that return their outputs."""
    z = _types(gen, 3000, 300, "outside", torch.int32)
    table, grad = _normal(gen, 300, 96, dtype=BF16), _normal(gen, 3000, 96, dtype=BF16)
    x, dd, post, g, scale, nxt = _norm_inputs(gen, 700, 160, "full", BF16)
    gy, gh = _normal(gen, 700, 160, dtype=BF16), _normal(gen, 700, 160, dtype=BF16)
    w, wt = ops.quantize(_normal(gen, 320, 160, dtype=BF16), columns=True)
    gw = _normal(gen, 700, 320, dtype=BF16)

    def train():
        y, xt = ops.block_linear(x, w, keep=True)
        return (y,) + ops.block_linear_gradient(gw, wt, xt)
    return [lambda: (ops.embed(z, table, 2.0),), lambda: (ops.embed_gradient(z, grad, 300, 2.0),),
            lambda: (ops.embed_gradient(z, grad, 4, 2.0),),
            lambda: ops.residual_norm(x, dd, post, g, scale, nxt),
            lambda: ops.residual_norm_gradient(x, dd, post, g, scale, nxt, gy, gh), train,
            lambda: (ops.block_linear(x[:3], w),),
            lambda: (ops.block_product(ops.norm(x, nxt, quantized=True), w, BF16),)]


def test_other_streams(gen):
    calls = _calls(gen)
    want = [f() for f in calls]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [f() for f in calls]
    side.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_graph_replays(gen):
    calls = _calls(gen)
    want = [f() for f in calls]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for f in calls:
            f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [f() for f in calls]
    for k in range(4):
        for a in got:
            for t in a:
                t.fill_(float(k))
        eager = [f() for f in calls]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b, e in zip(want, got, eager):
            assert all(torch.equal(s, t) and torch.equal(s, u) for s, t, u in zip(a, b, e))


def test_offsets_beyond_32_bits(gen):
    """Row strides that bring the last rows past 2^32 bytes (and 2^31 values)."""
    rows, stride = 40, (1 << 26) + 64
    room = torch.empty(rows * stride, dtype=BF16, device="cuda")

    def far(t):
        v = room.view(rows, stride)[:t.shape[0], :t.shape[1]]
        v.copy_(t)
        return v
    x = _normal(gen, rows, 300, dtype=BF16)
    z = torch.arange(rows, device="cuda")
    assert torch.equal(ops.embed(z, far(x)), x)
    assert torch.equal(ops.embed_gradient(z, far(x), rows), x)
    w = 1 + 0.1 * _normal(gen, 300)
    assert torch.equal(ops.norm(far(x), w), ops.norm(x, w))
    for a, b in zip(ops.residual_norm_gradient(far(x), None, None, None, None, w, x, x),
                    ops.residual_norm_gradient(x, None, None, None, None, w, x, x)):
        assert a is b is None or torch.equal(a, b)
    for a, b in zip(ops.quantize(far(x), columns=True), ops.quantize(x, columns=True)):
        assert torch.equal(a.values.view(torch.uint8), b.values.view(torch.uint8))


def test_last_byte_bounds():
    """The bounds above are those of the types."""
    assert UNIT[BF16] == torch.finfo(BF16).eps / 2 and LEAST[F16] == torch.finfo(F16).smallest_normal * 2.0 ** -10
