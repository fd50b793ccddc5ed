"""GPU tests of the gradients' norm and clipping against their definitions in float64."""

import math

import pytest
import torch

from _node_reference import assert_within, d
from symmetrix import node_ops as ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(13)


def _some(gen, sizes, dtypes, scale=1.0):
    return [(torch.randn(n, generator=gen, device="cuda") * scale).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def _norm(tensors):
    return math.sqrt(math.fsum(float(d(t).square().sum()) for t in tensors))


def _close(got, want):
    """One rounding to FP32; FP64 sums of fewer than 2^28 squares are off by 2^-25 of the result at the very most."""
    assert got.shape == () and got.dtype is F32
    assert abs(got.item() - want) <= (2.0 ** -24 + 2.0 ** -25) * want


SIZES = [[1], [0, 5], [7, 8, 9], [16383], [16384], [16385, 1], [100000, 3, 0, 77], [5] * 97, [1023] * 96, [33] * 300, [1 << 22, 11]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), s[0]))
@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F16], TYPES], ids=IDS + ["mixed"])
def test_norm_and_clipping(gen, sizes, dtypes):
    tensors = _some(gen, sizes, dtypes)
    want = _norm(tensors)
    _close(ops.gradient_norm(tensors), want)
    _close(ops.gradient_norm(tensors, scale=0.25), 0.25 * want)
    for most in (0.5 * want, 2.0 * want + 1.0):
        factor = min(1.0, most / want) if want else 1.0
        out = [torch.empty_like(t, dtype=TYPES[i % 3]) for i, t in enumerate(tensors)]
        _close(ops.clip_gradients(tensors, most, out=out), want)
        for t, o in zip(tensors, out):
            # the factor and the product are rounded to FP32, and max_norm to FP32 when it is handed over
            assert_within(o, d(t) * factor, 3 * 2.0 ** -24 * (d(t) * factor).abs() if factor < 1 else 0.0)
        held = [t.clone() for t in tensors]
        _close(ops.clip_gradients(held, most), want)
        for t, h in zip(tensors, held):
            assert_within(h, d(t) * factor, 3 * 2.0 ** -24 * (d(t) * factor).abs() if factor < 1 else 0.0)
            if factor == 1:
                assert torch.equal(t, h)


def test_scaled_loss(gen):
    """FP16 gradients of a loss that was scaled up: unscaled, clipped and brought to FP32 in one call."""
    tensors = _some(gen, [1000, 37], [F16], 30.0)
    want = _norm(tensors) / 1024
    out = [torch.empty_like(t, dtype=F32) for t in tensors]
    _close(ops.clip_gradients(tensors, 0.25, scale=1 / 1024, out=out), want)
    for t, o in zip(tensors, out):
        exact = d(t) / 1024 * 0.25 / want
        assert_within(o, exact, 2 * 2.0 ** -24 * exact.abs())


def test_shapes_orders_and_alignments(gen):
    base = torch.randn(50000, generator=gen, device="cuda")
    tensors = [base[1:].view(49999)[:20001], base[30000:30600].view(20, 30).t(), base[31001:31601].view(2, 10, 30).permute(2, 0, 1),
               torch.randn((), generator=gen, device="cuda"), torch.randn(3, 0, device="cuda")]
    want = _norm(tensors)
    _close(ops.gradient_norm(tensors), want)
    held = [t.clone() for t in tensors]
    ops.clip_gradients(tensors, 1.0)
    for a, b in zip(tensors, held):
        assert_within(a, d(b) / want, 2 * 2.0 ** -24 * (d(b) / want).abs())
    # (between them nothing is written)
    assert base[0] != 0 and torch.equal(base[20002:30000], torch.randn(50000, generator=torch.Generator(device="cuda").manual_seed(13),
                                                                       device="cuda")[20002:30000])


def test_large_and_small_values():
    """Squares beyond FP32, and a factor below its normal numbers."""
    t = torch.full((64,), 2.0 ** 127, device="cuda")
    assert ops.gradient_norm([t]).item() == math.inf  # 2^130: the norm is FP32
    assert ops.gradient_norm([t], scale=2.0 ** -30).item() == 2.0 ** 100
    ops.clip_gradients([t], 8.0)
    assert torch.equal(t, torch.ones_like(t))
    t = torch.full((1 << 18,), 3e38, device="cuda")
    ops.clip_gradients([t], 1.0)
    # 2^-9, to the rounding of the factor's significand and of the product
    assert ((t - 2.0 ** -9).abs() <= 2.0 ** -9 * 3 * 2.0 ** -24).all()
    small = torch.full((1024,), 2.0 ** -140, device="cuda")
    assert ops.gradient_norm([small]).item() == 2.0 ** -135
    zeros = torch.zeros(100, device="cuda")
    assert ops.clip_gradients([zeros], 0.0).item() == 0.0 and (zeros == 0).all()


def test_norms_that_are_no_numbers():
    t = [torch.ones(5, device="cuda"), torch.tensor([1.0, math.inf], device="cuda", dtype=BF16)]
    assert ops.clip_gradients(t, 1.0).item() == math.inf
    assert (t[0] == 0).all() and t[1][0] == 0 and torch.isnan(t[1][1])
    t = [torch.ones(5, device="cuda"), torch.tensor([1.0, math.nan], device="cuda", dtype=F16)]
    assert math.isnan(ops.clip_gradients(t, 1.0).item())
    assert all(torch.isnan(a).all() for a in t)
    t = [torch.tensor([3.0, 4.0], device="cuda")]
    assert ops.clip_gradients(t, math.inf).item() == 5.0 and t[0].tolist() == [3.0, 4.0]


def test_graph_and_stream(gen):
    sizes = [1000, 70000, 3]
    data = [_some(gen, sizes, TYPES, s) for s in (1.0, 1e-4, 100.0)]
    held = [t.clone() for t in data[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.clip_gradients(held, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_gradients(held, 1.0)
    for tensors in data:
        eager = [t.clone() for t in tensors]
        want = ops.clip_gradients(eager, 1.0)
        for a, b in zip(held, tensors):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(held, eager))


def test_beyond_32_bits(gen):
    t = torch.zeros((1 << 32) + 5, dtype=BF16, device="cuda")
    t[-3:] = 2.0
    t[0] = 2.0
    assert ops.gradient_norm([t]).item() == 4.0
    ops.clip_gradients([t], 2.0)
    assert t[-3:].tolist() == [1.0] * 3 and t[0] == 1.0 and t[1 << 31] == 0.0


def test_a_graph_notices_clipping(gen):
    """A tensor that a graph kept is not the one that it kept any more: going back through it is refused, as after torch's own
    changes in place."""
    w, g = torch.ones(50, device="cuda", requires_grad=True), torch.randn(50, generator=gen, device="cuda")
    for out in (None, [torch.empty_like(g)]):
        kept = g if out is None else out[0]
        y = (w * kept).sum()
        ops.gradient_norm([kept])
        y.backward(retain_graph=True)
        ops.clip_gradients([g], 0.5, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_lists_with_gaps(gen):
    """A parameter without a gradient has None, which is no tensor."""
    t = torch.randn(50, generator=gen, device="cuda")
    for call in (ops.gradient_norm, lambda ts: ops.clip_gradients(ts, 1.0), lambda ts: ops.clip_gradients([t, t], 1.0, out=ts)):
        for bad in (None, 1.0, t.double(), t.to_sparse()):
            with pytest.raises(ValueError, match="must be dense float32|must fill their memory"):
                call([t.clone(), bad])
