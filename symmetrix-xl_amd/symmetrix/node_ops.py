"""Node operators on torch tensors: what a learned block over an evaluator's atoms is made
of (include/symmetrix_node_ops.h).

* ``embed`` / ``embed_gradient``: scaled rows of a species table, and the
  table's gradient;
* ``norm``, ``residual_norm`` / ``residual_norm_gradient``: the norms before and
  after a block with its gate and residual scale;
* ``quantize``, ``block_product``, ``block_linear`` / ``block_linear_gradient``:
  products of E4M3 values with a power-of-two scale for each block of 128.

Row tensors are float32, bfloat16 or float16 on the current HIP device, two-dimensional, with
unit stride along the channels and any row stride.  Calls enqueue on torch's
current stream and return without waiting; a tensor made on another stream
is the caller's to order, as with torch's own operations.  Refused arguments raise
``ValueError`` before anything is launched.  The functions take and return plain values and record
nothing for autograd (``symmetrix.node_blocks`` wraps them).

torch brings a HIP runtime of its own, which this library shares when torch is
imported first; with two runtimes in the process a stream of one means nothing to the other, so
this module refuses to load then.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native
from ._native import check, lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_BLOCK = 128


def _one_runtime():
    try:
        with open("/proc/self/maps") as f:
            found = {line.split(None, 5)[5].strip() for line in f if "libamdhip64.so" in line}
    except OSError:
        return
    if len(found) > 1:
        raise ImportError("two HIP runtimes are loaded (%s): import torch before symmetrix to use symmetrix.node_ops"
                          % ", ".join(sorted(found)))


_one_runtime()


class BlockValues:
    """A matrix in 8-bit blocks along its rows: E4M3 ``values`` [rows][columns rounded up to
    128] and E8M0 ``scales`` (a byte for each block, four-aligned)."""

    __slots__ = ("values", "scales", "shape")

    def __init__(self, values, scales, shape):
        self.values, self.scales, self.shape = values, scales, shape

    def float(self):
        """The values that the blocks stand for, in float32."""
        r, c = self.shape
        blocks = -(-c // _BLOCK)
        v = self.values.to(torch.float32).reshape(r, blocks, _BLOCK)
        e = self.scales[:, :blocks].to(torch.int32) - 127
        return torch.ldexp(v, e[:, :, None]).reshape(r, blocks * _BLOCK)[:, :c]


def _stream(t):
    if not t.is_cuda:
        raise ValueError("node operators take tensors on a HIP device")
    if t.device.index != torch.cuda.current_device():
        raise ValueError("node operators take tensors of the current device")
    return torch.cuda.current_stream().cuda_stream


def _rows(t, name, like=None, channels=None, rows=None):
    """Checks a row tensor; its row stride in elements."""
    if t.dim() != 2:
        raise ValueError("%s must be two-dimensional" % name)
    if t.dtype not in _DTYPES:
        raise ValueError("%s must be float32, bfloat16 or float16" % name)
    if like is not None and (t.dtype is not like.dtype or t.device != like.device):
        raise ValueError("%s must have the type and device of the other rows" % name)
    r, c = t.shape
    if (channels is not None and c != channels) or (rows is not None and r != rows):
        raise ValueError("%s has the wrong shape" % name)
    stride, unit = t.stride()
    if (unit != 1 and c > 1) or (r > 1 and stride < c):
        raise ValueError("%s must have unit stride along its channels and rows that do not overlap" % name)
    return stride if r > 1 else max(stride, c)


def _vector(t, name, like, channels):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.device != like.device or t.shape != (channels,) or not t.is_contiguous():
        raise ValueError("%s must be a contiguous float32 vector of the channels, on the rows' device" % name)
    return t.data_ptr()


def _workspace(size, like):
    return torch.empty(size, dtype=torch.uint8, device=like.device) if size else None


def _at(t):
    return None if t is None else t.data_ptr()


# ---- species embedding ----


def _types(types, like):
    if types.dim() != 1 or types.dtype not in (torch.int32, torch.int64) or not types.is_contiguous() \
            or types.device != like.device:
        raise ValueError("types must be a contiguous int32 or int64 vector on the rows' device")
    return 1 if types.dtype is torch.int64 else 0


def embed(types, table, scale=1.0):
    """``scale * table[types]``; a type outside the table gives a row of zeros."""
    stride = _rows(table, "table")
    wide = _types(types, table)
    stream = _stream(table)
    t, (v, c) = types.shape[0], table.shape
    out = torch.empty((t, c), dtype=table.dtype, device=table.device)
    check(lib.smx_embed(types.data_ptr(), wide, t, table.data_ptr(), stride, v, c, _DTYPES[table.dtype], scale,
                        out.data_ptr(), c, stream))
    return out


def embed_gradient(types, grad, num_types, scale=1.0):
    """The table's gradient [num_types][channels]: for each type, ``scale`` times the sum of
    its atoms' rows of ``grad``, in a fixed order."""
    stride = _rows(grad, "grad", rows=types.shape[0])
    wide = _types(types, grad)
    stream = _stream(grad)
    t, c = grad.shape
    out = torch.empty((num_types, c), dtype=grad.dtype, device=grad.device)
    size = lib.smx_embed_gradient_workspace(t, num_types, c)
    room = _workspace(size, grad)
    check(lib.smx_embed_gradient(types.data_ptr(), wide, t, grad.data_ptr(), stride, num_types, c,
                                 _DTYPES[grad.dtype], scale, out.data_ptr(), c, _at(room), size, stream))
    return out


# ---- residual norm ----


def _gate(gate, x):
    """(kind, row stride) of the gate logits."""
    if gate is None:
        return 0, 0
    if gate.dtype is not x.dtype or gate.device != x.device:
        raise ValueError("gate must have the type and device of the rows")
    r, c = x.shape
    if gate.dim() == 1 and gate.shape[0] == c:
        if c > 1 and gate.stride(0) != 1:
            raise ValueError("a channel gate must be contiguous")
        return 2, 0
    if gate.dim() == 2 and gate.shape == (r, c) and c > 1:
        return 1, _rows(gate, "gate", x)
    if gate.dim() == 2 and gate.shape == (r, 1):
        if r > 1 and gate.stride(0) < 1:
            raise ValueError("the rows of a gate must not overlap")
        return 3, max(gate.stride(0), 1)
    raise ValueError("gate must be [rows][channels], [channels] or [rows][1]")


def _norm_args(x, d, post, gate, scale, next_weight, eps):
    xs = _rows(x, "x")
    r, c = x.shape
    if d is None:
        if gate is not None or post is not None or scale is not None:
            raise ValueError("post, gate and scale go with d")
        ds, kind, gs = 0, 0, 0
    else:
        ds = _rows(d, "d", x, c, r)
        if post is None:
            raise ValueError("post must be given with d")
        kind, gs = _gate(gate, x)
    a = _native.SmxResidualNormArgs(
        ctypes.sizeof(_native.SmxResidualNormArgs), _DTYPES[x.dtype], r, c, x.data_ptr(), xs, _at(d), ds, _at(gate), gs,
        kind, eps, _vector(post, "post", x, c), _vector(scale, "scale", x, c), _vector(next_weight, "next_weight", x, c))
    return a


def residual_norm(x, d, post, gate=None, scale=None, next_weight=None, eps=1e-6, quantized=False):
    """``(y, h)``: ``y = x + scale * sigmoid(gate) * post * d / rms(d)`` and, with ``next_weight``,
    ``h = next_weight * y / rms(y)`` (else None), as ``BlockValues`` when ``quantized``.

    ``gate``: logits, one for each value ([rows][channels]), channel ([channels]) or row
    ([rows][1]); ``post``, ``scale`` and ``next_weight``: float32 [channels]."""
    a = _norm_args(x, d, post, gate, scale, next_weight, eps)
    stream = _stream(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = _norm_outputs(a, x, y, next_weight, quantized)
    check(lib.smx_residual_norm(ctypes.byref(a), stream))
    return y, h


def norm(x, weight, eps=1e-6, quantized=False):
    """``weight * x / rms(x)``, as ``BlockValues`` when ``quantized``."""
    a = _norm_args(x, None, None, None, None, weight, eps)
    stream = _stream(x)
    h = _norm_outputs(a, x, None, weight, quantized)
    check(lib.smx_residual_norm(ctypes.byref(a), stream))
    return h


def _norm_outputs(a, x, y, next_weight, quantized):
    r, c = x.shape
    if y is not None:
        a.y, a.y_stride = y.data_ptr(), c
    if next_weight is None:
        return None
    if not quantized:
        h = torch.empty((r, c), dtype=x.dtype, device=x.device)
        a.h, a.h_stride = h.data_ptr(), c
        return h
    h = _empty_blocks(r, c, x.device)
    a.h, a.h_scales = h.values.data_ptr(), h.scales.data_ptr()
    return h


def residual_norm_gradient(x, d, post, gate, scale, next_weight, grad_y, grad_h, eps=1e-6):
    """Gradients ``(x, d, gate, post, scale, next_weight)`` of ``residual_norm`` from its inputs
    and the gradients of ``y`` and ``h`` (either may be None); None for inputs that are None.
    Those of ``post``, ``scale`` and ``next_weight`` are float32."""
    a = _norm_args(x, d, post, gate, scale, next_weight, eps)
    r, c = x.shape
    g = _native.SmxResidualNormGradientArgs(a)
    if grad_y is not None:
        g.grad_y_stride = _rows(grad_y, "grad_y", x, c, r)
        g.grad_y = grad_y.data_ptr()
    if grad_h is not None:
        if next_weight is None:
            raise ValueError("grad_h without next_weight")
        g.grad_h_stride = _rows(grad_h, "grad_h", x, c, r)
        g.grad_h = grad_h.data_ptr()
    stream = _stream(x)
    dx = torch.empty((r, c), dtype=x.dtype, device=x.device)
    g.dx, g.dx_stride = dx.data_ptr(), c
    dd = dg = dpost = dscale = dnext = None
    # the channel vectors' gradients share one allocation
    vectors = torch.empty((3, c), dtype=torch.float32, device=x.device)
    if d is not None:
        dd = torch.empty((r, c), dtype=x.dtype, device=x.device)
        g.dd, g.dd_stride = dd.data_ptr(), c
        dpost = vectors[0]
        g.dpost = dpost.data_ptr()
        if scale is not None:
            dscale = vectors[1]
            g.dscale = dscale.data_ptr()
        if gate is not None:
            dg = torch.empty(gate.shape, dtype=x.dtype, device=x.device)
            g.dgate, g.dgate_stride = dg.data_ptr(), gate.shape[-1]
    if next_weight is not None:
        dnext = vectors[2]
        g.dnext = dnext.data_ptr()
    size = lib.smx_residual_norm_gradient_workspace(r, c)
    room = _workspace(size, x)
    g.workspace, g.workspace_bytes = _at(room), size
    check(lib.smx_residual_norm_gradient(ctypes.byref(g), stream))
    return dx, dd, dg, dpost, dscale, dnext


# ---- 8-bit block product ----


def _empty_blocks(rows, cols, device):
    pitch = -(-cols // _BLOCK) * _BLOCK
    blocks = pitch // _BLOCK
    return BlockValues(torch.empty((rows, pitch), dtype=torch.float8_e4m3fn, device=device),
                       torch.empty((rows, -(-blocks // 4) * 4), dtype=torch.uint8, device=device), (rows, cols))


def quantize(x, rows=True, columns=False):
    """``x`` in 8-bit blocks along its rows, or (``columns``) its transpose in blocks along
    x's columns; both, in one pass, as a pair."""
    stride = _rows(x, "x")
    if not (rows or columns):
        raise ValueError("neither rows nor columns are asked for")
    stream = _stream(x)
    r, c = x.shape
    a = _empty_blocks(r, c, x.device) if rows else None
    b = _empty_blocks(c, r, x.device) if columns else None
    check(lib.smx_block_quantize(x.data_ptr(), stride, _DTYPES[x.dtype], r, c, _at(a and a.values),
                                 _at(a and a.scales), _at(b and b.values), _at(b and b.scales), stream))
    return (a, b) if rows and columns else a if rows else b


def _check_blocks(b, name, k, device):
    if not isinstance(b, BlockValues):
        raise ValueError("%s must be BlockValues (symmetrix.node_ops.quantize)" % name)
    if b.shape[1] != k or b.values.device != device:
        raise ValueError("%s must have as many columns as the other operand, on its device" % name)


def _product_dtype(dtype):
    if dtype not in _DTYPES:
        raise ValueError("products are float32, bfloat16 or float16")
    return _DTYPES[dtype]


def block_product(a, b, dtype=torch.float32):
    """``a @ b.T`` of two ``BlockValues``, [m][k] and [n][k]."""
    if not isinstance(a, BlockValues):
        raise ValueError("a must be BlockValues (symmetrix.node_ops.quantize)")
    (m, k), n = a.shape, b.shape[0]
    device = a.values.device
    _check_blocks(b, "b", k, device)
    code = _product_dtype(dtype)
    stream = _stream(a.values)
    out = torch.empty((m, n), dtype=dtype, device=device)
    size = lib.smx_block_product_workspace(m, n, k)
    room = _workspace(size, a.values)
    check(lib.smx_block_product(_at(a.values), _at(a.scales), _at(b.values), _at(b.scales), m, n, k, code,
                                out.data_ptr(), n, _at(room), size, stream))
    return out


def block_linear(x, w, dtype=None, keep=False):
    """``x @ w.T`` with x [m][k] brought to 8-bit blocks within the call and ``w`` the weights'
    ``BlockValues`` [n][k]; in x's type unless ``dtype`` is given.  With ``keep`` the pair of the
    product and x's column blocks, which ``block_linear_gradient`` takes."""
    stride = _rows(x, "x")
    m, k = x.shape
    _check_blocks(w, "w", k, x.device)
    if dtype is None:
        dtype = x.dtype
    if keep:
        rows, columns = quantize(x, columns=True)
        return block_product(rows, w, dtype), columns
    code = _product_dtype(dtype)
    stream = _stream(x)
    n = w.shape[0]
    out = torch.empty((m, n), dtype=dtype, device=x.device)
    size = lib.smx_block_linear_workspace(m, n, k)
    room = _workspace(size, x)
    check(lib.smx_block_linear(x.data_ptr(), stride, _DTYPES[x.dtype], _at(w.values), _at(w.scales), m, n, k, code,
                               out.data_ptr(), n, _at(room), size, stream))
    return out


def block_linear_gradient(grad, w_columns, x_columns, dtype=None):
    """``(dx, dw)`` of ``y = x @ w.T`` from y's gradient [m][n]: ``grad @ w`` in grad's type and
    ``grad.T @ x`` in float32 (``dtype``), each a product of 8-bit blocks along its own summed axis.

    ``w_columns``: the weights' column blocks (``quantize(w, columns=True)[1]``), ``x_columns``
    those that ``block_linear(..., keep=True)`` gave; None leaves that gradient out."""
    if w_columns is None and x_columns is None:
        return None, None
    both = quantize(grad, rows=w_columns is not None, columns=x_columns is not None)
    rows, columns = both if isinstance(both, tuple) else (both, both)
    dx = None if w_columns is None else block_product(rows, w_columns, grad.dtype)
    dw = None if x_columns is None else block_product(columns, x_columns, dtype or torch.float32)
    return dx, dw


__all__ = ["BlockValues", "embed", "embed_gradient", "norm", "residual_norm", "residual_norm_gradient", "quantize",
           "block_product", "block_linear", "block_linear_gradient"]
