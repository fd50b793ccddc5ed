"""CPU tests of refusals by the operators of rows by type, of clipping and of integers: in Python before any
allocation or launch, and at the C boundary before any launch (pointers here are never read)."""

import copy
import ctypes
import math
import pickle

import pytest
import torch

from symmetrix import node_ops
from symmetrix._native import SMX_ERR_INVALID_ARGUMENT, SMX_ERR_UNSUPPORTED, SymmetrixUnsupportedError, lib

P = 1 << 20  # an address that nothing reads


def _groups(rows, v):
    return node_ops.RowGroups(rows, v, torch.zeros(lib.smx_group_plan_bytes(rows, v) // 4, dtype=torch.int32))


def _integers(r, c):
    return node_ops.IntegerValues(torch.zeros(r, -(-c // 128) * 128, dtype=torch.int8), torch.zeros(r), (r, c))


def _bad(rc, text, code=SMX_ERR_INVALID_ARGUMENT):
    assert rc == code and text in lib.smx_last_error().decode(), (rc, lib.smx_last_error())


# ---- rows by type ----


def test_group_rows():
    z = torch.zeros(5, dtype=torch.int64)
    for bad in (torch.zeros(5), torch.zeros(5, 1, dtype=torch.int64), torch.zeros(10, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="int32 or int64 vector"):
            node_ops.group_rows(bad, 4)
    with pytest.raises(ValueError, match="positive"):
        node_ops.group_rows(z, 0)
    with pytest.raises(SymmetrixUnsupportedError, match="4096"):
        node_ops.group_rows(z, 4097)
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.group_rows(z, 4)
    for f in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="group_rows"):
            f(_groups(5, 4))


def test_plan_sizes():
    assert lib.smx_group_plan_bytes(-1, 4) == lib.smx_group_plan_bytes(3, 0) == lib.smx_group_plan_bytes(3, 4097) == 0
    for v in (1, 2, 3, 89, 4096):
        order = lib.smx_group_plan_order(v)
        assert order % 16 == 0 and order >= 16 + 4 * (v + 1) and lib.smx_group_plan_bytes(7, v) == order + 28
        g = _groups(7, v)
        assert g.offsets.shape == (v + 1,) and g.order.shape == (7,)


def test_group_rows_at_the_boundary():
    size = lib.smx_group_plan_bytes(5000, 4)
    work = lib.smx_group_rows_workspace(5000, 4)
    assert work > 0

    def call(types=P, wide=0, rows=5000, v=4, plan=P, size=size, room=P, work=work):
        return lib.smx_group_rows(types, wide, rows, v, plan, size, room, work, None)
    _bad(call(types=None), "types is NULL")
    _bad(call(types=P + 4, wide=1), "not aligned")
    _bad(call(rows=-1), "rows must be")
    _bad(call(rows=(1 << 30) + 1), "rows must be")
    _bad(call(v=0), "a kind at least")
    _bad(call(v=4097), "4096", SMX_ERR_UNSUPPORTED)
    _bad(call(plan=None), "the plan is NULL")
    _bad(call(plan=P + 8), "16-byte")
    _bad(call(size=size - 1), "too small")
    _bad(call(room=None), "workspace")
    _bad(call(work=work - 1), "workspace")


def test_grouped_linear():
    x, grad, w, g = torch.zeros(5, 8), torch.zeros(5, 6), torch.zeros(3, 6, 8), _groups(5, 3)
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.grouped_linear(x, w, g)
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.grouped_linear_gradient(grad, x, w, g)
    cases = [((x, w, None), "RowGroups"), ((x[:4], w, g), "rows that were grouped"), ((x.double(), w, g), "float32, bfloat16"),
             ((x[0], w, g), "two-dimensional"), ((x.t().contiguous().t(), w, g), "unit stride"), ((x, w.half(), g), "type and device"),
             ((x, w[:2], g), "types"), ((x, w[0], g), "types"), ((x, torch.zeros(3, 6, 9), g), "inputs"),
             ((x, torch.zeros(3, 8, 6).transpose(1, 2), g), "unit stride"), ((x, w[:1].expand(3, 6, 8), g), "overlap"),
             ((x, torch.zeros(3, 1, 8).expand(3, 6, 8), g), "do not overlap"), ((x, w, g, torch.float16), "rows' type or float32"),
             ((x, w, g, torch.float64), "rows' type or float32")]
    for args, text in cases:
        with pytest.raises(ValueError, match=text):
            node_ops.grouped_linear(*args)
    cases = [((grad[:4], x, w, g), "rows that were grouped"), ((grad, x[:4], w, g), "rows that were grouped"),
             ((grad, x.half(), w, g), "type and device"), ((grad, x, torch.zeros(3, 7, 8), g), "outputs"),
             ((grad, x, torch.zeros(3, 6, 9), g), "inputs"), ((grad, x, w, None), "RowGroups"),
             ((grad, x, w, g, torch.bfloat16), "rows' type or float32")]
    for args, text in cases:
        with pytest.raises(ValueError, match=text):
            node_ops.grouped_linear_gradient(*args)


def test_grouped_linear_at_the_boundary():
    def forward(x=P, xs=8, dt=1, w=P, ws=8, wt=48, plan=P, rows=5, v=3, k=8, n=6, odt=1, out=P, os=6):
        return lib.smx_grouped_linear(x, xs, dt, w, ws, wt, plan, rows, v, k, n, odt, out, os, None)

    def by_rows(x=P, xs=6, dt=1, w=P, ws=8, wt=48, plan=P, rows=5, v=3, k=8, n=6, odt=1, out=P, os=8):
        return lib.smx_grouped_linear_by_rows(x, xs, dt, w, ws, wt, plan, rows, v, k, n, odt, out, os, None)
    for call, name, result in ((forward, "x", "out"), (by_rows, "grad", "dx")):
        _bad(call(x=None), "%s is NULL" % name)
        _bad(call(x=P + 1), "%s is not aligned" % name)
        _bad(call(xs=5), "%s: the row stride" % name)
        _bad(call(dt=7), "unknown dtype")
        _bad(call(odt=2), "rows' type or FP32")
        _bad(call(w=None), "w is NULL")
        _bad(call(ws=7), "w: the row stride")
        _bad(call(wt=47), "two kinds overlap")
        _bad(call(plan=None), "the plan")
        _bad(call(plan=P + 4), "the plan")
        _bad(call(rows=-1), "rows must be")
        _bad(call(v=0), "a kind at least")
        _bad(call(v=5000), "4096", SMX_ERR_UNSUPPORTED)
        _bad(call(k=-1), "inputs must be")
        _bad(call(n=(1 << 24) + 1), "outputs must be")
        _bad(call(out=None), "%s is NULL" % result)
        _bad(call(os=5), "%s: the row stride" % result)
        assert call(rows=0, x=None, out=None) == 0

    size = lib.smx_grouped_linear_by_weights_workspace(5000, 3, 8, 6)
    assert size > 0 and size % 16 == 0 and lib.smx_grouped_linear_by_weights_workspace(0, 3, 8, 6) == 0

    def by_weights(g=P, gs=6, x=P, xs=8, dt=1, plan=P, rows=5000, v=3, k=8, n=6, odt=0, dw=P, ws=8, wt=48, room=P, size=size):
        return lib.smx_grouped_linear_by_weights(g, gs, x, xs, dt, plan, rows, v, k, n, odt, dw, ws, wt, room, size, None)
    _bad(by_weights(g=None), "grad is NULL")
    _bad(by_weights(x=None), "x is NULL")
    _bad(by_weights(dw=None), "dw is NULL")
    _bad(by_weights(wt=40), "two kinds overlap")
    _bad(by_weights(odt=2), "rows' type or FP32")
    _bad(by_weights(room=None), "workspace")
    _bad(by_weights(size=size - 1), "workspace")
    _bad(by_weights(room=P + 8), "16-byte")


# ---- clipping ----


def test_clip_gradients():
    a, b = torch.ones(4), torch.ones(3, 5)
    for f in (node_ops.gradient_norm, lambda t: node_ops.clip_gradients(t, 1.0)):
        with pytest.raises(ValueError, match="HIP device"):
            f([a, b])
        with pytest.raises(ValueError, match="none"):
            f([])
        with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
            f([a, b.double()])
        with pytest.raises(ValueError, match="without gaps"):
            f([torch.ones(4, 6)[:, :5]])
        with pytest.raises(ValueError, match="without gaps"):
            f([torch.ones(1, 5).expand(4, 5)])
    for out, text in (([a], "as many"), ([b, a], "shapes"), ([a.clone(), torch.ones(5, 3).t()], "strides"),
                      ([a.clone(), b.int()], "float32, bfloat16 or float16")):
        with pytest.raises(ValueError, match=text):
            node_ops.clip_gradients([a, b], 1.0, out=out)
    with pytest.raises(ValueError, match="detach"):
        node_ops.clip_gradients([a, b.clone().requires_grad_()], 1.0)
    with pytest.raises(ValueError, match="detach"):
        node_ops.clip_gradients([a], 1.0, out=[a.clone().requires_grad_()])
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.clip_gradients([a.clone().requires_grad_()], 1.0, out=[a])


def test_clipping_at_the_boundary():
    def call(at=(P, P + 4096), counts=(10, 20), codes=(0, 1), n=None, most=1.0, scale=1.0, out=None, out_codes=None, norm=P, room=P,
             size=lib.smx_gradient_norm_workspace(), clip=True):
        n = len(at) if n is None else n
        out, out_codes = at if out is None else out, codes if out_codes is None else out_codes
        a, c, t = (ctypes.c_void_p * len(at))(*at), (ctypes.c_int64 * len(counts))(*counts), (ctypes.c_int32 * len(codes))(*codes)
        if not clip:
            return lib.smx_gradient_norm(a, c, t, n, scale, norm, room, size, None)
        return lib.smx_clip_gradients(a, c, t, n, most, scale, (ctypes.c_void_p * len(out))(*out),
                                      (ctypes.c_int32 * len(out_codes))(*out_codes), norm, room, size, None)
    for clip in (False, True):
        _bad(call(n=-1, clip=clip), "number of tensors")
        _bad(call(at=(None, P), clip=clip), "a tensor is NULL")
        _bad(call(at=(P + 2, P + 4096), clip=clip), "not aligned")
        _bad(call(counts=(-1, 3), clip=clip), "count")
        _bad(call(codes=(0, 3), clip=clip), "unknown dtype")
        _bad(call(norm=None, clip=clip), "norm is NULL")
        _bad(call(room=None, clip=clip), "workspace")
        _bad(call(size=8, clip=clip), "workspace")
        for scale in (0.0, -1.0, math.inf, math.nan):
            _bad(call(scale=scale, clip=clip), "scale must be")
    for most in (-1.0, math.nan):
        _bad(call(most=most), "max_norm")
    _bad(call(out=(P + (1 << 16), None)), "an output is NULL")
    _bad(call(out=(P + (1 << 16), P + (1 << 16) + 36)), "two outputs overlap")
    _bad(call(at=(P, P)), "two outputs overlap")
    _bad(call(out=(P + 4096, P)), "not its own")
    _bad(call(out=(P + 4, P + 8192)), "not its own")
    _bad(call(out_codes=(1, 1)), "not its own")
    many = 98305
    _bad(call(at=(P,) * many, counts=(1,) * many, codes=(0,) * many, clip=False), "98304", SMX_ERR_UNSUPPORTED)


# ---- integers ----


def test_integers():
    x, w = torch.zeros(4, 8), _integers(6, 8)
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.quantize_integers(x)
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.integer_linear(x, w)
    with pytest.raises(ValueError, match="HIP device"):
        node_ops.integer_product(_integers(4, 8), w)
    for f, text in ((lambda: node_ops.quantize_integers(x.double()), "float32, bfloat16"),
                    (lambda: node_ops.quantize_integers(x[0]), "two-dimensional"),
                    (lambda: node_ops.integer_linear(x, x), "IntegerValues"),
                    (lambda: node_ops.integer_linear(x, _integers(6, 9)), "as many columns"),
                    (lambda: node_ops.integer_linear(x, w, torch.int32), "products are"),
                    (lambda: node_ops.integer_product(x, w), "IntegerValues"),
                    (lambda: node_ops.integer_product(_integers(4, 9), w), "as many columns"),
                    (lambda: node_ops.integer_product(_integers(4, 8), w, torch.float64), "products are")):
        with pytest.raises(ValueError, match=text):
            f()
    values, scales = torch.zeros(6, 128, dtype=torch.int8), torch.zeros(6)
    for args, text in (((values.to(torch.uint8), scales, (6, 8)), "int8"), ((values, scales, (6, 129)), "values"),
                       ((values.t().contiguous().t(), scales, (6, 8)), "contiguous"), ((values, scales.double(), (6, 8)), "scales"),
                       ((values, torch.zeros(5), (6, 8)), "scales"), ((values, torch.zeros(12)[::2], (6, 8)), "scales")):
        with pytest.raises(ValueError, match=text):
            node_ops.IntegerValues(*args)
    for name in ("values", "scales", "shape"):
        with pytest.raises(AttributeError):
            setattr(w, name, None)
    for name in ("rows", "num_types", "order", "offsets"):
        with pytest.raises(AttributeError):
            setattr(_groups(5, 3), name, None)
    back = pickle.loads(pickle.dumps(w))
    assert back.shape == w.shape and torch.equal(back.values, w.values)


def test_integers_at_the_boundary():
    assert [lib.smx_integer_stride(c) for c in (-1, 0, 1, 128, 129)] == [0, 0, 128, 128, 256]

    def quantize(x=P, xs=8, dt=1, rows=4, cols=8, values=P, scales=P):
        return lib.smx_integer_quantize(x, xs, dt, rows, cols, values, scales, None)
    _bad(quantize(x=None), "x is NULL")
    _bad(quantize(xs=7), "row stride")
    _bad(quantize(dt=-1), "unknown dtype")
    _bad(quantize(rows=-1), "sizes")
    _bad(quantize(cols=-1), "sizes")
    _bad(quantize(values=None), "values is NULL")
    _bad(quantize(scales=None), "values is NULL")
    _bad(quantize(values=P + 8), "16-byte")

    def product(a=P, sa=P, b=P, sb=P, m=4, n=6, k=8, dt=1, out=P, os=6):
        return lib.smx_integer_product(a, sa, b, sb, m, n, k, dt, out, os, None)
    _bad(product(a=None), "a is NULL")
    _bad(product(sb=None), "b is NULL")
    _bad(product(b=P + 4), "16-byte")
    _bad(product(out=None), "out is NULL")
    _bad(product(os=5), "row stride")
    _bad(product(dt=5), "unknown dtype")
    _bad(product(m=-1), "sizes")
    _bad(product(k=(1 << 17) + 1), "2^17", SMX_ERR_UNSUPPORTED)
    assert product(m=0, a=None, sa=None, out=None) == 0

    size = lib.smx_integer_linear_workspace(40, 6, 8)
    assert size == 40 * 128 + 160 and lib.smx_integer_linear_workspace(0, 6, 8) == 0

    def linear(x=P, xs=8, dt=1, w=P, sw=P, m=40, n=6, k=8, odt=1, out=P, os=6, room=P, size=size):
        return lib.smx_integer_linear(x, xs, dt, w, sw, m, n, k, odt, out, os, room, size, None)
    _bad(linear(x=None), "x is NULL")
    _bad(linear(w=None), "w is NULL")
    _bad(linear(odt=9), "unknown dtype")
    _bad(linear(room=None), "workspace")
    _bad(linear(size=size - 1), "workspace")
    _bad(linear(k=(1 << 17) + 1, xs=1 << 18), "2^17", SMX_ERR_UNSUPPORTED)
