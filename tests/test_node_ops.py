"""CPU tests of the node operators: what the C entry points and the Python functions refuse (before any
device work), the sizes they report, and the float64 reference against autograd and differences."""

import ctypes
import math

import pytest
import torch

from _node_reference import Norm, quantized
from symmetrix import _native, node_ops

lib = _native.lib
FAKE = 1 << 20  # an aligned address that no refused call may touch
INVALID, UNSUPPORTED = _native.SMX_ERR_INVALID_ARGUMENT, _native.SMX_ERR_UNSUPPORTED


def _refused(rc, text, code=INVALID):
    assert rc == code
    assert text in lib.smx_last_error().decode()


def test_embed_refuses():
    def call(types=FAKE, tokens=4, table=FAKE, stride=8, v=3, c=8, dtype=0, out=FAKE, out_stride=8):
        return lib.smx_embed(types, 0, tokens, table, stride, v, c, dtype, 1.0, out, out_stride, None)
    _refused(call(types=None), "types is NULL")
    _refused(call(types=FAKE + 2), "types is not aligned")
    _refused(call(tokens=-1), "tokens")
    _refused(call(tokens=1 << 31), "tokens")
    _refused(call(v=-1), "num_types")
    _refused(call(c=1 << 31), "channels")
    _refused(call(dtype=3), "dtype")
    _refused(call(dtype=-1), "dtype")
    _refused(call(table=None), "table is NULL")
    _refused(call(stride=7), "table: the row stride")
    _refused(call(out_stride=7), "out: the row stride")
    _refused(call(out=FAKE + 2), "out is not aligned")
    assert call(tokens=0, types=None, out=None) == 0


def test_embed_gradient_refuses():
    def call(types=FAKE, tokens=100, grad=FAKE, stride=8, v=3, c=8, out=FAKE, room=FAKE, size=None):
        size = lib.smx_embed_gradient_workspace(tokens, v, c) if size is None else size
        return lib.smx_embed_gradient(types, 1, tokens, grad, stride, v, c, 1, 1.0, out, 8, room, size, None)
    _refused(call(types=None), "types is NULL")
    _refused(call(types=FAKE + 4), "types is not aligned")  # int64 here
    _refused(call(grad=None), "grad is NULL")
    _refused(call(stride=4), "grad: the row stride")
    _refused(call(out=None), "out is NULL")
    assert lib.smx_embed_gradient_workspace(256, 3, 8) == 0  # few atoms need none
    assert lib.smx_embed_gradient_workspace(5000, 3, 8) > 0
    _refused(call(tokens=5000, size=0), "workspace")
    _refused(call(tokens=5000, room=None), "workspace")
    _refused(call(tokens=5000, room=FAKE + 8), "aligned")
    assert call(v=0, out=None) == 0


def _norm_args(**more):
    a = _native.SmxResidualNormArgs(ctypes.sizeof(_native.SmxResidualNormArgs), 0, 4, 16, FAKE, 16, FAKE, 16, FAKE, 16,
                                    1, 1e-6, FAKE, FAKE, FAKE, FAKE, 16, FAKE, 16, None)
    for k, v in more.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change, text", [
    ({"struct_size": 8}, "struct_size"), ({"dtype": 7}, "dtype"), ({"rows": -1}, "rows"), ({"rows": 1 << 31}, "rows"),
    ({"channels": 0}, "channels"), ({"x": None}, "x is NULL"), ({"x_stride": 15}, "x: the row stride"),
    ({"d_stride": 3}, "d: the row stride"), ({"post": None}, "post is NULL"), ({"gate_kind": 4}, "gate kind"),
    ({"gate": None}, "gate is NULL"), ({"gate_stride": 1}, "gate: the row stride"),
    ({"gate": None, "gate_kind": 3}, "gate is NULL"), ({"next": None}, "without next"), ({"h": None}, "h is NULL"),
    ({"y_stride": 8}, "y: the row stride"), ({"h_stride": 8}, "h: the row stride"), ({"eps": -1.0}, "eps"),
    ({"h_scales": FAKE + 4}, "16-byte"), ({"y": None, "h": None, "next": None}, "neither"),
    ({"post": FAKE + 2}, "aligned"), ({"y": FAKE + 1}, "aligned")])
def test_residual_norm_refuses(change, text):
    _refused(lib.smx_residual_norm(ctypes.byref(_norm_args(**change)), None), text)


def test_residual_norm_unsupported_and_empty():
    wide = _norm_args(channels=16385, x_stride=20000, d_stride=20000, gate_stride=20000, y_stride=20000, h_stride=20000)
    _refused(lib.smx_residual_norm(ctypes.byref(wide), None), "16384", UNSUPPORTED)
    _refused(lib.smx_residual_norm(None, None), "NULL")
    assert lib.smx_residual_norm(ctypes.byref(_norm_args(rows=0, x=None, d=None, y=None, h=None)), None) == 0


@pytest.mark.parametrize("change, text", [
    ({"grad_y_stride": 3}, "grad_y: the row stride"), ({"grad_h_stride": 3}, "grad_h: the row stride"),
    ({"dx_stride": 3}, "dx: the row stride"), ({"dd_stride": 3}, "dd: the row stride"),
    ({"dgate_stride": 3}, "dgate: the row stride"), ({"workspace_bytes": 0}, "workspace"),
    ({"workspace": FAKE + 4}, "aligned")])
def test_residual_norm_gradient_refuses(change, text):
    def args(a):
        size = lib.smx_residual_norm_gradient_workspace(4, 16)
        g = _native.SmxResidualNormGradientArgs(a, FAKE, 16, FAKE, 16, FAKE, 16, FAKE, 16, FAKE, 16, FAKE, FAKE, FAKE,
                                                FAKE, size)
        for k, v in change.items():
            setattr(g, k, v)
        return ctypes.byref(g)
    _refused(lib.smx_residual_norm_gradient(args(_norm_args()), None), text)


def test_residual_norm_gradient_refuses_outputs_without_inputs():
    def rc(a, **outs):
        g = _native.SmxResidualNormGradientArgs(a, FAKE, 16, None, 0)
        g.workspace, g.workspace_bytes = FAKE, 1 << 20
        for k, v in outs.items():
            setattr(g, k, v)
        return lib.smx_residual_norm_gradient(ctypes.byref(g), None)
    _refused(rc(_norm_args(d=None), dd=FAKE, dd_stride=16), "without d")
    _refused(rc(_norm_args(gate_kind=0), dgate=FAKE, dgate_stride=16), "without a gate")
    _refused(rc(_norm_args(scale=None), dscale=FAKE), "without scale")
    _refused(rc(_norm_args(next=None), dnext=FAKE), "without next")
    _refused(rc(_norm_args(next=None), grad_h=FAKE, grad_h_stride=16), "without next")
    _refused(lib.smx_residual_norm_gradient(None, None), "NULL")


def test_block_sizes():
    assert [lib.smx_block_stride(k) for k in (-3, 0, 1, 128, 129, 1000)] == [0, 0, 128, 128, 256, 1024]
    assert [lib.smx_block_scale_stride(k) for k in (-3, 0, 1, 512, 513, 1025)] == [0, 0, 4, 4, 8, 12]


def test_block_quantize_refuses():
    def call(x=FAKE, stride=8, dtype=0, rows=4, cols=8, v=FAKE, s=FAKE, vt=None, st=None):
        return lib.smx_block_quantize(x, stride, dtype, rows, cols, v, s, vt, st, None)
    _refused(call(x=None), "x is NULL")
    _refused(call(stride=5), "row stride")
    _refused(call(dtype=9), "dtype")
    _refused(call(rows=-1), "sizes")
    _refused(call(s=None), "go together")
    _refused(call(st=FAKE), "go together")
    _refused(call(v=None, s=None), "no output")
    _refused(call(v=FAKE + 8), "16-byte")
    assert call(rows=0, x=None, v=None, s=None) == 0


def test_block_product_refuses():
    def call(a=FAKE, sa=FAKE, b=FAKE, sb=FAKE, m=4, n=8, k=16, dtype=0, out=FAKE, stride=8, room=FAKE, size=None):
        size = lib.smx_block_product_workspace(m, n, k) if size is None else size
        return lib.smx_block_product(a, sa, b, sb, m, n, k, dtype, out, stride, room, size, None)
    _refused(call(a=None), "a is NULL")
    _refused(call(sb=None), "b is NULL")
    _refused(call(b=FAKE + 4), "16-byte")
    _refused(call(m=-1), "sizes")
    _refused(call(k=1 << 31), "sizes")
    _refused(call(dtype=5), "dtype")
    _refused(call(out=None), "out is NULL")
    _refused(call(stride=7), "row stride")
    assert call(m=0, a=None, sa=None, out=None) == 0


def test_block_linear_refuses():
    def call(x=FAKE, xs=16, dtype=0, w=FAKE, ws=FAKE, m=40, n=8, k=16, od=1, out=FAKE, stride=8, room=FAKE, size=None):
        size = lib.smx_block_linear_workspace(m, n, k) if size is None else size
        return lib.smx_block_linear(x, xs, dtype, w, ws, m, n, k, od, out, stride, room, size, None)
    _refused(call(x=None), "x is NULL")
    _refused(call(xs=15), "x: the row stride")
    _refused(call(dtype=4), "dtype")
    _refused(call(od=4), "dtype")
    _refused(call(w=None), "w is NULL")
    _refused(call(out=FAKE + 1), "aligned")
    _refused(call(size=0), "workspace")
    _refused(call(n=-8), "sizes")
    assert call(m=0, x=None, out=None) == 0


def test_python_refusals():
    x = torch.zeros(4, 8)
    z = torch.zeros(4, dtype=torch.int32)
    one = torch.ones(8)
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.embed(z, x)
    with pytest.raises(ValueError, match="two-dimensional"):
        node_ops.embed(z, x[0])
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        node_ops.embed(z, x.double())
    with pytest.raises(ValueError, match="int32 or int64"):
        node_ops.embed(z.float(), x)
    with pytest.raises(ValueError, match="int32 or int64"):
        node_ops.embed(torch.zeros(8, dtype=torch.int32)[::2], x)
    with pytest.raises(ValueError, match="unit stride"):
        node_ops.embed(z, x.T)
    with pytest.raises(ValueError, match="unit stride"):
        node_ops.quantize(one.expand(4, 8))
    with pytest.raises(ValueError, match="wrong shape"):
        node_ops.embed_gradient(z[:3], x, 5)
    with pytest.raises(ValueError, match="go with d"):
        node_ops.residual_norm(x, None, one)
    with pytest.raises(ValueError, match="post must be given"):
        node_ops.residual_norm(x, x, None)
    with pytest.raises(ValueError, match="float32 vector"):
        node_ops.residual_norm(x, x, one[:7])
    with pytest.raises(ValueError, match="float32 vector"):
        node_ops.norm(x, one.bfloat16())
    with pytest.raises(ValueError, match="gate must be"):
        node_ops.residual_norm(x, x, one, torch.zeros(4))
    with pytest.raises(ValueError, match="type and device"):
        node_ops.residual_norm(x, x.bfloat16(), one)
    with pytest.raises(ValueError, match="grad_h without"):
        node_ops.residual_norm_gradient(x, x, one, None, None, None, x, x)
    with pytest.raises(ValueError, match="neither"):
        node_ops.quantize(x, rows=False)
    with pytest.raises(ValueError, match="BlockValues"):
        node_ops.block_linear(x, x)
    def bytes_of(*shape):
        return torch.zeros(*shape, dtype=torch.uint8)
    blocks = node_ops.BlockValues(bytes_of(3, 128), bytes_of(3, 4), (3, 9))
    with pytest.raises(ValueError, match="as many columns"):
        node_ops.block_linear(x, blocks)
    with pytest.raises(ValueError, match="as many columns"):
        node_ops.block_product(node_ops.BlockValues(bytes_of(3, 128), bytes_of(3, 4), (3, 8)), blocks)
    with pytest.raises(ValueError, match="products are"):
        node_ops.block_product(blocks, blocks, torch.float64)
    for values, scales, shape in ((bytes_of(3, 127), bytes_of(3, 4), (3, 9)), (bytes_of(3, 128), bytes_of(3, 1), (3, 9)),
                                  (bytes_of(3, 128), bytes_of(3, 4), (3, 129)), (bytes_of(2, 128), bytes_of(3, 4), (3, 9)),
                                  (torch.zeros(3, 128), bytes_of(3, 4), (3, 9)),
                                  (bytes_of(128, 3).T, bytes_of(3, 4), (3, 9))):
        with pytest.raises(ValueError, match="contiguous bytes"):
            node_ops.BlockValues(values, scales, shape)


# ---- the reference itself ----


def test_quantized_reference():
    x = torch.zeros(1, 6, dtype=torch.float64)
    x[0] = torch.tensor([448.0, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, math.inf])
    q, byte = quantized(x)
    assert byte.tolist() == [[127]]  # 448 fits a scale of one
    # ties to even: 1.0625 -> 1, 1.1875 -> 1.25; half of the least subnormal 2^-9 -> 0, three halves -> 2 of them
    assert q[0, :5].tolist() == [448.0, 1.0, 1.25, 0.0, 2.0 ** -8]
    assert math.isnan(q[0, 5])
    assert quantized(x[:, :1] * 1.0000001)[1].tolist() == [[128]]
    assert quantized(x[:, :1] * 0)[1].tolist() == [[0]]


@pytest.mark.parametrize("gate", ["none", "full", "channel", "row"])
def test_norm_reference_gradients(gate):
    g = torch.Generator().manual_seed(5)
    r, c = 3, 7

    def n(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    leaves = {"x": n(r, c), "d": n(r, c), "post": n(c), "scale": n(c), "next": n(c)}
    shape = {"full": (r, c), "channel": (c,), "row": (r, 1)}.get(gate)
    if shape:
        leaves["gate"] = n(*shape)
    gy, gh = n(r, c), n(r, c)

    def loss(v):
        f = Norm(v["x"], v["d"], v["post"], v.get("gate"), v["scale"], v["next"], 1e-6)
        return (f.y * gy + f.h * gh).sum().item()
    got, _ = Norm(leaves["x"], leaves["d"], leaves["post"], leaves.get("gate"), leaves["scale"], leaves["next"],
                  1e-6).backward(gy, gh)
    for name, t in leaves.items():
        way = n(*t.shape)
        h = 1e-5
        up, down = ({**leaves, name: t + s * h * way} for s in (1, -1))
        # central differences: O(h^2) of the third derivative and 1e-16 / h of rounding
        assert abs((loss(up) - loss(down)) / (2 * h) - (got[name] * way).sum().item()) < 1e-6
