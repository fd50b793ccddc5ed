"""Node operators on torch tensors: what a learned block over an evaluator's atoms is made
of (include/symmetrix_node_ops.h).

* ``embed`` / ``embed_gradient``: scaled rows of a species table, and the
  table's gradient;
* ``norm``, ``residual_norm`` / ``residual_norm_gradient``: the norms before and
  after a block with its gate and residual scale;
* ``quantize``, ``block_product``, ``block_linear`` / ``block_linear_gradient``:
  products of E4M3 values with a power-of-two scale for each block of 128;
* ``group_rows``, ``grouped_linear`` / ``grouped_linear_gradient``: rows by their
  type, products with a weight matrix for each type, and their gradients;
* ``gradient_norm``, ``clip_gradients``: the norm of many gradients together, and
  their clipping;
* ``quantize_integers``, ``integer_product``, ``integer_linear``: products of 8-bit
  integers with a scale for each row of both operands.

Row tensors are float32, bfloat16 or float16 on the current HIP device, two-dimensional, with
unit stride along the channels and any row stride.  Calls enqueue on torch's
current stream and return without waiting; a tensor made on another stream
is the caller's to order, as with torch's own operations.  Refused arguments raise
``ValueError`` before anything is launched, and sizes that an operator has no kernel for
``SymmetrixUnsupportedError`` before it launches.  The functions take and return plain values and record
nothing for autograd (``symmetrix.node_blocks`` wraps them).

torch brings a HIP runtime of its own, which this library shares when torch is
imported first; with two runtimes in the process a stream of one means nothing to the other, so
this module refuses to load then.
"""

from __future__ import annotations

import array
import ctypes
import functools
import operator

import torch

from . import _native
from ._native import SymmetrixUnsupportedError, check, lib

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
    128] and E8M0 ``scales`` (a byte for each block, four-aligned).  Either may be given as uint8;
    ``values`` is float8_e4m3fn and ``scales`` uint8 however they were.  Copies (``copy``, ``pickle``,
    ``torch.save`` and ``torch.load``) are made of these tensors and checked like new ones."""

    __slots__ = ("shape", "_room")

    def __init__(self, values, scales, shape):
        rows, cols = shape
        pitch, scale_pitch = _pitches(cols)
        for t, name, width, kind in ((values, "values", pitch, torch.float8_e4m3fn),
                                     (scales, "scales", scale_pitch, torch.float8_e8m0fnu)):
            if t.dtype not in (torch.uint8, kind) or tuple(t.shape) != (rows, width) or not t.is_contiguous() \
                    or t.data_ptr() % 16:
                raise ValueError("%s must be contiguous bytes (uint8 or %s) [%d][%d], 16-byte aligned"
                                 % (name, str(kind).replace("torch.", ""), rows, width))
        if values.device != scales.device:
            raise ValueError("values and scales must be on one device")
        values, scales = values.view(torch.float8_e4m3fn), scales.view(torch.uint8)
        self.shape, self._room = (rows, cols), (values, scales)

    @classmethod
    def _empty(cls, rows, cols, like):
        """Room for a matrix: values and then scales in one allocation."""
        self = cls.__new__(cls)
        pitch, scale_pitch = _pitches(cols)
        room = torch.empty(rows * (pitch + scale_pitch), dtype=torch.uint8, device=like.device)
        self.shape, self._room = (rows, cols), room
        return self

    @property
    def _at(self):
        """The addresses of values and scales, of the tensors as they are at each call."""
        if isinstance(self._room, tuple):
            return self._room[0].data_ptr(), self._room[1].data_ptr()
        at = self._room.data_ptr()
        return at, at + self.shape[0] * _pitches(self.shape[1])[0]

    def __reduce__(self):
        # (as uint8, which every way of saving a tensor takes)
        return BlockValues, (self.values.view(torch.uint8), self.scales, self.shape)

    def _split(self):
        if not isinstance(self._room, tuple):
            rows, cols = self.shape
            pitch, scale_pitch = _pitches(cols)
            self._room = (self._room[:rows * pitch].view(torch.float8_e4m3fn).view(rows, pitch),
                          self._room[rows * pitch:].view(rows, scale_pitch))
        return self._room

    @property
    def values(self):
        return self._split()[0]

    @property
    def scales(self):
        return self._split()[1]

    def _device(self):
        return (self._room[0] if isinstance(self._room, tuple) else self._room).get_device()

    def float(self):
        """The values that the blocks stand for, in float32."""
        r, c = self.shape
        blocks = -(-c // _BLOCK)
        v = self.values.to(torch.float32).reshape(r, blocks, _BLOCK)
        e = self.scales[:, :blocks].to(torch.int32) - 127
        return torch.ldexp(v, e[:, :, None]).reshape(r, blocks * _BLOCK)[:, :c]


def _pitches(cols):
    blocks = -(-cols // _BLOCK)
    return blocks * _BLOCK, -(-blocks // 4) * 4


# so that torch.load, which by default makes only what it knows to be safe, makes them too
torch.serialization.add_safe_globals([BlockValues])

# the current stream's handle without the Stream object around it, which costs more than some of the calls here
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream(device):
    if device < 0:
        raise ValueError("node operators take tensors on a HIP device")
    if device != torch.cuda.current_device():
        raise ValueError("node operators take tensors of the current device")
    return _raw_stream(device)


def _rows(t, name):
    """Checks a row tensor; (type code, rows, channels, row stride in elements)."""
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError("%s must be float32, bfloat16 or float16" % name)
    shape = t.shape
    if len(shape) != 2:
        raise ValueError("%s must be two-dimensional" % name)
    r, c = shape
    stride, unit = t.stride()
    if (unit != 1 and c > 1) or (stride < c and r > 1):
        raise ValueError("%s must have unit stride along its channels and rows that do not overlap" % name)
    return code, r, c, stride if r > 1 else c


def _like(t, name, x, shape):
    """Checks another row tensor of x's type and device; its row stride in elements."""
    if t.dtype is not x.dtype or t.get_device() != x.get_device():
        raise ValueError("%s must have the type and device of the other rows" % name)
    if t.shape != shape:
        raise ValueError("%s has the wrong shape" % name)
    return _rows(t, name)[3]


def _vector(t, name, device, channels):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.dim() != 1 or t.numel() != channels or t.get_device() != device \
            or not t.is_contiguous():
        raise ValueError("%s must be a contiguous float32 vector of the channels, on the rows' device" % name)
    return t.data_ptr()


def _same(x):
    """Room for rows like x's, packed."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _workspace(size, like):
    return torch.empty(size, dtype=torch.uint8, device=like.device) if size else None


def _at(t):
    return None if t is None else t.data_ptr()


# ---- species embedding ----


def _types(types, like):
    wide = types.dtype is torch.int64
    if (not wide and types.dtype is not torch.int32) or types.dim() != 1 or not types.is_contiguous() \
            or types.get_device() != like.get_device():
        raise ValueError("types must be a contiguous int32 or int64 vector on the rows' device")
    return wide


def embed(types, table, scale=1.0):
    """``scale * table[types]``; a type outside the table gives a row of zeros."""
    code, v, c, stride = _rows(table, "table")
    wide = _types(types, table)
    stream = _stream(table.get_device())
    t = types.shape[0]
    out = table.new_empty((t, c))
    check(lib.smx_embed(types.data_ptr(), wide, t, table.data_ptr(), stride, v, c, code, scale, out.data_ptr(), c,
                        stream))
    return out


def embed_gradient(types, grad, num_types, scale=1.0):
    """The table's gradient [num_types][channels]: for each type, ``scale`` times the sum of
    its atoms' rows of ``grad``, in a fixed order."""
    code, t, c, stride = _rows(grad, "grad")
    wide = _types(types, grad)
    if types.shape[0] != t:
        raise ValueError("grad has the wrong shape")
    if num_types < 0:
        raise ValueError("num_types must not be negative")
    stream = _stream(grad.get_device())
    out = grad.new_empty((num_types, c))
    size = lib.smx_embed_gradient_workspace(t, num_types, c)
    room = _workspace(size, grad)
    check(lib.smx_embed_gradient(types.data_ptr(), wide, t, grad.data_ptr(), stride, num_types, c, code, scale,
                                 out.data_ptr(), c, _at(room), size, stream))
    return out


# ---- residual norm ----


def _gate(gate, x, shape):
    """(kind, row stride) of the gate logits."""
    if gate.dtype is not x.dtype or gate.get_device() != x.get_device():
        raise ValueError("gate must have the type and device of the rows")
    r, c = shape
    given = gate.shape
    if len(given) == 2 and given == shape and c > 1:
        return 1, _rows(gate, "gate")[3]
    if len(given) == 1 and given[0] == c:
        if c > 1 and gate.stride(0) != 1:
            raise ValueError("a channel gate must be contiguous")
        return 2, 0
    if len(given) == 2 and given == (r, 1):
        if r > 1 and gate.stride(0) < 1:
            raise ValueError("the rows of a gate must not overlap")
        return 3, max(gate.stride(0), 1)
    raise ValueError("gate must be [rows][channels], [channels] or [rows][1]")


_NORM_ARGS = ctypes.sizeof(_native.SmxResidualNormArgs)


def _norm_inputs(x, d, post, gate, scale, next_weight, eps):
    """Checks; the fields of SmxResidualNormArgs up to its outputs."""
    code, r, c, xs = _rows(x, "x")
    device = x.get_device()
    if d is None:
        if gate is not None or post is not None or scale is not None:
            raise ValueError("post, gate and scale go with d")
        return (_NORM_ARGS, code, r, c, x.data_ptr(), xs, None, 0, None, 0, 0, eps, None, None,
                _vector(next_weight, "next_weight", device, c))
    shape = x.shape
    ds = _like(d, "d", x, shape)
    if post is None:
        raise ValueError("post must be given with d")
    if gate is None:
        kind, at, gs = 0, None, 0
    else:
        kind, gs = _gate(gate, x, shape)
        at = gate.data_ptr()
    return (_NORM_ARGS, code, r, c, x.data_ptr(), xs, d.data_ptr(), ds, at, gs, kind, eps,
            _vector(post, "post", device, c), _vector(scale, "scale", device, c),
            _vector(next_weight, "next_weight", device, c))


def residual_norm(x, d, post, gate=None, scale=None, next_weight=None, eps=1e-6, quantized=False):
    """``(y, h)``: ``y = x + scale * sigmoid(gate) * post * d / rms(d)`` and, with ``next_weight``,
    ``h = next_weight * y / rms(y)`` (else None), as ``BlockValues`` when ``quantized``.

    ``gate``: logits, one for each value ([rows][channels]), channel ([channels]) or row
    ([rows][1]); ``post``, ``scale`` and ``next_weight``: float32 [channels]."""
    inputs = _norm_inputs(x, d, post, gate, scale, next_weight, eps)
    stream = _stream(x.get_device())
    c = inputs[3]
    y = _same(x)
    h, at, scales = (None, None, None) if next_weight is None else _norm_output(x, quantized)
    rc = lib.smx_residual_norm(_native.SmxResidualNormArgs(*inputs, y.data_ptr(), c, at, c, scales), stream)
    if rc:
        check(rc)
    return y, h


def norm(x, weight, eps=1e-6, quantized=False):
    """``weight * x / rms(x)``, as ``BlockValues`` when ``quantized``."""
    inputs = _norm_inputs(x, None, None, None, None, weight, eps)
    stream = _stream(x.get_device())
    c = inputs[3]
    h, at, scales = _norm_output(x, quantized)
    rc = lib.smx_residual_norm(_native.SmxResidualNormArgs(*inputs, None, 0, at, c, scales), stream)
    if rc:
        check(rc)
    return h


def _norm_output(x, quantized):
    """(h, its address, its scales' address)"""
    if quantized:
        h = BlockValues._empty(x.shape[0], x.shape[1], x)
        return (h, *h._at)
    h = _same(x)
    return h, h.data_ptr(), None


def residual_norm_gradient(x, d, post, gate, scale, next_weight, grad_y, grad_h, eps=1e-6):
    """Gradients ``(x, d, gate, post, scale, next_weight)`` of ``residual_norm`` from its inputs
    and the gradients of ``y`` and ``h`` (either may be None); None for inputs that are None.
    Those of ``post``, ``scale`` and ``next_weight`` are float32."""
    inputs = _norm_inputs(x, d, post, gate, scale, next_weight, eps)
    r, c, shape = inputs[2], inputs[3], x.shape
    gys = ghs = 0
    if grad_y is not None:
        gys = _like(grad_y, "grad_y", x, shape)
    if grad_h is not None:
        if next_weight is None:
            raise ValueError("grad_h without next_weight")
        ghs = _like(grad_h, "grad_h", x, shape)
    stream = _stream(x.get_device())
    dx = _same(x)
    dd = dg = dpost = dscale = dnext = None
    if d is not None:
        dd, dpost = _same(x), torch.empty_like(post)
        if scale is not None:
            dscale = torch.empty_like(scale)
        if gate is not None:
            dg = _same(gate)
    if next_weight is not None:
        dnext = torch.empty_like(next_weight)
    size = lib.smx_residual_norm_gradient_workspace(r, c)
    room = _workspace(size, x)
    g = _native.SmxResidualNormGradientArgs(
        _native.SmxResidualNormArgs(*inputs), _at(grad_y), gys, _at(grad_h), ghs, dx.data_ptr(), c, _at(dd), c, _at(dg),
        1 if inputs[10] == 3 else c, _at(dpost), _at(dscale), _at(dnext), _at(room), size)
    rc = lib.smx_residual_norm_gradient(g, stream)
    if rc:
        check(rc)
    return dx, dd, dg, dpost, dscale, dnext


# ---- 8-bit block product ----


def quantize(x, rows=True, columns=False):
    """``x`` in 8-bit blocks along its rows, or (``columns``) its transpose in blocks along
    x's columns; both, in one pass, as a pair."""
    code, r, c, stride = _rows(x, "x")
    if not (rows or columns):
        raise ValueError("neither rows nor columns are asked for")
    stream = _stream(x.get_device())
    a = BlockValues._empty(r, c, x) if rows else None
    b = BlockValues._empty(c, r, x) if columns else None
    av, asc = a._at if rows else (None, None)
    bv, bsc = b._at if columns else (None, None)
    check(lib.smx_block_quantize(x.data_ptr(), stride, code, r, c, av, asc, bv, bsc, stream))
    return (a, b) if rows and columns else a if rows else b


def _check_blocks(b, name, k, device):
    if not isinstance(b, BlockValues):
        raise ValueError("%s must be BlockValues (symmetrix.node_ops.quantize)" % name)
    if b.shape[1] != k or b._device() != device:
        raise ValueError("%s must have as many columns as the other operand, on its device" % name)


def _product_dtype(dtype):
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError("products are float32, bfloat16 or float16")
    return code


def block_product(a, b, dtype=torch.float32):
    """``a @ b.T`` of two ``BlockValues``, [m][k] and [n][k]."""
    if not isinstance(a, BlockValues):
        raise ValueError("a must be BlockValues (symmetrix.node_ops.quantize)")
    m, k = a.shape
    device = a._device()
    _check_blocks(b, "b", k, device)
    n = b.shape[0]
    code = _product_dtype(dtype)
    stream = _stream(device)
    out = torch.empty((m, n), dtype=dtype, device=device)
    size = lib.smx_block_product_workspace(m, n, k)
    room = _workspace(size, out)
    check(lib.smx_block_product(*a._at, *b._at, m, n, k, code, out.data_ptr(), n, _at(room), size, stream))
    return out


def block_linear(x, w, dtype=None, keep=False):
    """``x @ w.T`` with x [m][k] brought to 8-bit blocks within the call and ``w`` the weights'
    ``BlockValues`` [n][k]; in x's type unless ``dtype`` is given.  With ``keep`` the pair of the
    product and x's column blocks, which ``block_linear_gradient`` takes."""
    code, m, k, stride = _rows(x, "x")
    device = x.get_device()
    _check_blocks(w, "w", k, device)
    out_code = code if dtype is None else _product_dtype(dtype)
    if keep:
        rows, columns = quantize(x, columns=True)
        return block_product(rows, w, x.dtype if dtype is None else dtype), columns
    current = _stream(device)
    n = w.shape[0]
    out = x.new_empty((m, n)) if dtype is None else x.new_empty((m, n), dtype=dtype)
    size = lib.smx_block_linear_workspace(m, n, k)
    room = _workspace(size, x)
    check(lib.smx_block_linear(x.data_ptr(), stride, code, *w._at, m, n, k, out_code, out.data_ptr(), n, _at(room), size,
                               current))
    return out


def block_linear_gradient(grad, w_columns, x_columns, dtype=None):
    """``(dx, dw)`` of ``y = x @ w.T`` from y's gradient [m][n]: ``grad @ w`` in grad's type and
    ``grad.T @ x`` in float32 (``dtype``), each a product of 8-bit blocks along its own summed axis.

    ``w_columns``: the weights' column blocks (``quantize(w, columns=True)[1]``), ``x_columns``
    those that ``block_linear(..., keep=True)`` gave; None leaves that gradient out."""
    _, m, n, _ = _rows(grad, "grad")
    for blocks, name, k in ((w_columns, "w_columns", n), (x_columns, "x_columns", m)):
        if blocks is not None:
            _check_blocks(blocks, name, k, grad.get_device())
    dw_dtype = torch.float32 if dtype is None else dtype
    _product_dtype(dw_dtype)
    if w_columns is None and x_columns is None:
        return None, None
    both = quantize(grad, rows=w_columns is not None, columns=x_columns is not None)
    rows, columns = both if isinstance(both, tuple) else (both, both)
    dx = None if w_columns is None else block_product(rows, w_columns, grad.dtype)
    dw = None if x_columns is None else block_product(columns, x_columns, dw_dtype)
    return dx, dw


# ---- rows by type ----


class RowGroups:
    """Rows in the order of their types (``group_rows``): ``order`` int32 [rows], by type, of one type as they come, masked
    ones last; ``offsets`` int32 [num_types + 1], where each type's rows begin in it.  Both lie on the device and are what the
    products read: they are not to be written to."""

    __slots__ = ("_rows", "_num_types", "_room")

    def __init__(self, rows, num_types, room):
        self._rows, self._num_types, self._room = rows, num_types, room

    rows = property(lambda self: self._rows)
    num_types = property(lambda self: self._num_types)

    @property
    def offsets(self):
        return self._room[4:5 + self._num_types]

    @property
    def order(self):
        return self._room[_plan_order(self._num_types) // 4:]

    def __reduce__(self):
        raise TypeError("RowGroups are not copied: make them of the types again (symmetrix.node_ops.group_rows)")


def _size(function):
    """A library function of sizes alone, whose answers are kept: the call costs as much as an allocation."""
    return functools.lru_cache(maxsize=1024)(lambda *sizes: function(*sizes))


_plan_order = _size(lib.smx_group_plan_order)
_group_room, _weights_room, _integer_room = (_size(f) for f in (
    lib.smx_group_rows_workspace, lib.smx_grouped_linear_by_weights_workspace, lib.smx_integer_linear_workspace))


def group_rows(types, num_types):
    """``RowGroups`` of ``types`` (a contiguous int32 or int64 vector); a type outside [0, num_types) masks its row."""
    wide = _types(types, types)
    if num_types < 1:
        raise ValueError("num_types must be positive")
    if num_types > 4096:
        raise SymmetrixUnsupportedError("rows are grouped by up to 4096 types")
    stream = _stream(types.get_device())
    t = types.shape[0]
    size = _plan_order(num_types) + 4 * t
    plan = torch.empty(size // 4, dtype=torch.int32, device=types.device)
    work = _group_room(t, num_types)
    room = _workspace(work, types)
    check(lib.smx_group_rows(types.data_ptr(), wide, t, num_types, plan.data_ptr(), size, _at(room), work, stream))
    return RowGroups(t, num_types, plan)


def _grouped(t, name, groups):
    """Checks rows of groups; (type code, channels, row stride)."""
    if not isinstance(groups, RowGroups):
        raise ValueError("groups must be RowGroups (symmetrix.node_ops.group_rows)")
    code, r, c, stride = _rows(t, name)
    if r != groups.rows or groups._room.get_device() != t.get_device():
        raise ValueError("%s must have the rows that were grouped, on their device" % name)
    return code, c, stride


def _type_weights(w, like, num_types, outputs, inputs):
    """Checks weights [num_types][outputs][inputs]; (row stride, type stride)."""
    if w.dtype is not like.dtype or w.get_device() != like.get_device():
        raise ValueError("w must have the type and device of the rows")
    if w.dim() != 3 or w.shape[0] != num_types or (outputs is not None and w.shape[1] != outputs) \
            or (inputs is not None and w.shape[2] != inputs):
        raise ValueError("w must be [types][outputs][inputs] of the grouped types and the rows' channels")
    v, n, k = w.shape
    by_type, by_row, unit = w.stride()
    if (unit != 1 and k > 1) or (by_row < k and n > 1):
        raise ValueError("w must have unit stride along its inputs and rows that do not overlap")
    if n <= 1:
        by_row = k
    if v > 1 and by_type < (n - 1) * by_row + k and n and k:
        raise ValueError("the types' matrices in w must not overlap")
    return by_row, by_type if v > 1 else n * by_row


def _out_dtype(dtype, like):
    if dtype is None or dtype is like.dtype:
        return like.dtype
    if dtype is not torch.float32:
        raise ValueError("products by type are of the rows' type or float32")
    return dtype


def grouped_linear(x, w, groups, dtype=None):
    """Each row of ``x`` [rows][inputs] through its type's matrix of ``w`` [num_types][outputs][inputs]; a masked row gives
    zeros.  Sums are FP32; in x's type unless ``dtype`` is float32."""
    code, k, xs = _grouped(x, "x", groups)
    ws, wt = _type_weights(w, x, groups.num_types, None, k)
    dtype = _out_dtype(dtype, x)
    stream = _stream(x.get_device())
    n = w.shape[1]
    out = torch.empty((groups.rows, n), dtype=dtype, device=x.device)
    rc = lib.smx_grouped_linear(x.data_ptr(), xs, code, w.data_ptr(), ws, wt, groups._room.data_ptr(), groups.rows,
                                groups.num_types, k, n, _DTYPES[dtype], out.data_ptr(), n, stream)
    if rc:
        check(rc)
    return out


def grouped_linear_gradient(grad, x, w, groups, dtype=None):
    """``(dx, dw)`` of ``grouped_linear`` from the gradient [rows][outputs] of its result: dx in grad's type (None where ``w`` is
    None) and dw [num_types][outputs][inputs] in float32, or ``dtype`` (None where ``x`` is None).  A type without rows
    has a gradient of zeros."""
    code, n, gs = _grouped(grad, "grad", groups)
    v, rows, plan = groups.num_types, groups.rows, groups._room.data_ptr()
    if x is not None:
        if x.dtype is not grad.dtype:
            raise ValueError("x must have the type and device of grad")
        _, k, xs = _grouped(x, "x", groups)
    if w is not None:
        ws, wt = _type_weights(w, grad, v, n, None if x is None else k)
    dw_dtype = _out_dtype(torch.float32 if dtype is None else dtype, grad)
    stream = _stream(grad.get_device())
    dx = dw = None
    if w is not None:
        dx = grad.new_empty((rows, w.shape[2]))
        check(lib.smx_grouped_linear_by_rows(grad.data_ptr(), gs, code, w.data_ptr(), ws, wt, plan, rows, v, w.shape[2], n,
                                             code, dx.data_ptr(), w.shape[2], stream))
    if x is not None:
        dw = torch.empty((v, n, k), dtype=dw_dtype, device=grad.device)
        size = _weights_room(rows, v, k, n)
        room = _workspace(size, grad)
        check(lib.smx_grouped_linear_by_weights(grad.data_ptr(), gs, x.data_ptr(), xs, code, plan, rows, v, k, n,
                                                _DTYPES[dw_dtype], dw.data_ptr(), k, n * k, _at(room), size, stream))
    return dx, dw


# ---- gradients' norm and clipping ----


def _packed(t):
    """Whether t's values fill one piece of memory, in whatever order of its axes."""
    if t.layout is not torch.strided:
        return False
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride != at:
            return False
        at *= size
    return True


def _axes(t):
    """The sizes and strides of t's axes, of those along which there is anything to step."""
    return [(n, s) for n, s in zip(t.shape, t.stride()) if n > 1]


_dtypes_of, _needs_grad = operator.attrgetter("dtype"), operator.attrgetter("requires_grad")
_T = torch.Tensor


def _table(tensors, name):
    """(addresses, counts, type codes, device, whether all are contiguous) of tensors, for the length of a call.  One pass of a
    built-in over all of them for each: a loop over them in Python took longer than the kernels for a small head's."""
    try:
        codes = array.array("i", map(_DTYPES.__getitem__, map(_dtypes_of, tensors)))
        packed = all(map(_T.is_contiguous, tensors))
    except (AttributeError, KeyError, RuntimeError, TypeError):
        raise ValueError("%s must be dense float32, bfloat16 or float16 tensors" % name) from None
    devices = set(map(_T.get_device, tensors))
    if len(devices) != 1:
        raise ValueError("%s must be on one device" % name)
    if not packed and not all(map(_packed, tensors)):
        raise ValueError("%s must fill their memory without gaps or overlaps" % name)
    return array.array("Q", map(_T.data_ptr, tensors)), array.array("q", map(_T.numel, tensors)), codes, devices.pop(), \
        packed


def _of(a):
    return a.buffer_info()[0]


_NORM_ROOM = lib.smx_gradient_norm_workspace()


def _norm_room(like):
    return (torch.empty((), dtype=torch.float32, device=like.device),
            torch.empty(_NORM_ROOM, dtype=torch.uint8, device=like.device), _NORM_ROOM)


def _listed(tensors, name):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise ValueError("%s are none" % name)
    return tensors


def gradient_norm(tensors, scale=1.0):
    """``scale`` times the 2-norm of all values of ``tensors`` together, a float32 scalar on their device.  The tensors are
    float32, bfloat16 or float16, in any mix, and fill their memory without gaps."""
    tensors = _listed(tensors, "tensors")
    at, counts, codes, device, _ = _table(tensors, "tensors")
    stream = _stream(device)
    norm, room, size = _norm_room(tensors[0])
    check(lib.smx_gradient_norm(_of(at), _of(counts), _of(codes), len(tensors), scale, norm.data_ptr(), room.data_ptr(), size,
                                stream))
    return norm


def clip_gradients(tensors, max_norm, scale=1.0, out=None):
    """Brings ``tensors`` to a norm of ``max_norm`` at most: each becomes ``tensor * scale * min(1, max_norm / norm)``, in place or
    in ``out`` (tensors of as many values each, in the same order, of any of the types).  The norm before it, ``scale`` times the
    2-norm of all values (``scale`` of gradients whose loss was scaled, 1 / the loss's), is returned as a float32 scalar on
    their device; nothing waits for it.  An infinite ``max_norm`` clips nothing, an infinite norm included.  Changed tensors do not ask
    for gradients themselves, and a graph that kept one refuses to go back through it."""
    tensors = _listed(tensors, "tensors")
    at, counts, codes, device, packed = _table(tensors, "tensors")
    to, to_codes = at, codes
    if out is not None:
        out = _listed(out, "out")
        if len(out) != len(tensors):
            raise ValueError("out must be as many tensors")
        to, to_counts, to_codes, to_device, to_packed = _table(out, "out")
        if to_device != device:
            raise ValueError("out must be on the tensors' device")
        if to_counts != counts:
            raise ValueError("out must have the tensors' shapes")
        # (contiguous ones of as many values hold them in one order)
        if not (packed and to_packed) and any(_axes(a) != _axes(b) for a, b in zip(tensors, out)
                                              if not (a.is_contiguous() and b.is_contiguous())):
            raise ValueError("out must have the tensors' shapes and strides")
    if any(map(_needs_grad, tensors if out is None else out)):
        raise ValueError("tensors that are changed must not ask for gradients themselves: detach them")
    stream = _stream(device)
    norm, room, size = _norm_room(tensors[0])
    check(lib.smx_clip_gradients(_of(at), _of(counts), _of(codes), len(tensors), max_norm, scale, _of(to), _of(to_codes),
                                 norm.data_ptr(), room.data_ptr(), size, stream))
    # (a refused call has changed nothing)
    torch.autograd.graph.increment_version(tensors if out is None else out)
    return norm


# ---- products in 8-bit integers ----


class IntegerValues:
    """A matrix in 8-bit integers: int8 ``values`` [rows][columns rounded up to 128, the rest zeros] and a float32 scale for each row,
    ``scales`` [rows].  Copies (``copy``, ``pickle``, ``torch.save`` and ``torch.load``) are made of these tensors and
    checked like new ones."""

    __slots__ = ("_shape", "_values", "_scales")

    def __init__(self, values, scales, shape):
        rows, cols = shape
        pitch = -(-cols // 128) * 128
        if values.dtype is not torch.int8 or tuple(values.shape) != (rows, pitch) or not values.is_contiguous() \
                or values.data_ptr() % 16:
            raise ValueError("values must be contiguous int8 [%d][%d], 16-byte aligned" % (rows, pitch))
        if scales.dtype is not torch.float32 or tuple(scales.shape) != (rows,) or not scales.is_contiguous():
            raise ValueError("scales must be contiguous float32 [%d]" % rows)
        if values.device != scales.device:
            raise ValueError("values and scales must be on one device")
        self._shape, self._values, self._scales = (rows, cols), values, scales

    shape = property(lambda self: self._shape)
    values = property(lambda self: self._values)
    scales = property(lambda self: self._scales)

    def __reduce__(self):
        return IntegerValues, (self.values, self.scales, self.shape)

    def float(self):
        """The values that the integers stand for, in float32."""
        return self.values[:, :self.shape[1]].to(torch.float32) * self.scales[:, None]


torch.serialization.add_safe_globals([IntegerValues])


def quantize_integers(x):
    """``x`` in 8-bit integers: for each row the whole numbers nearest to its values' quotients by a scale, the FP32 product of
    the largest magnitude and the FP32 number next to 1/127."""
    code, r, c, stride = _rows(x, "x")
    stream = _stream(x.get_device())
    out = IntegerValues.__new__(IntegerValues)
    out._shape = (r, c)
    out._values = torch.empty((r, -(-c // 128) * 128), dtype=torch.int8, device=x.device)
    out._scales = torch.empty(r, dtype=torch.float32, device=x.device)
    check(lib.smx_integer_quantize(x.data_ptr(), stride, code, r, c, out._values.data_ptr(), out._scales.data_ptr(), stream))
    return out


def _check_integers(b, name, k, device):
    if not isinstance(b, IntegerValues):
        raise ValueError("%s must be IntegerValues (symmetrix.node_ops.quantize_integers)" % name)
    if b.shape[1] != k or b.values.get_device() != device:
        raise ValueError("%s must have as many columns as the other operand, on its device" % name)


def integer_product(a, b, dtype=torch.float32):
    """``a @ b.T`` of two ``IntegerValues``, [m][k] and [n][k]; the sums are exact."""
    if not isinstance(a, IntegerValues):
        raise ValueError("a must be IntegerValues (symmetrix.node_ops.quantize_integers)")
    m, k = a.shape
    device = a.values.get_device()
    _check_integers(b, "b", k, device)
    n = b.shape[0]
    code = _product_dtype(dtype)
    stream = _stream(device)
    out = torch.empty((m, n), dtype=dtype, device=a.values.device)
    check(lib.smx_integer_product(a.values.data_ptr(), a.scales.data_ptr(), b.values.data_ptr(), b.scales.data_ptr(), m, n, k,
                                  code, out.data_ptr(), n, stream))
    return out


def integer_linear(x, w, dtype=None):
    """``x @ w.T`` with x [m][k] brought to 8-bit integers within the call and ``w`` the weights' ``IntegerValues`` [n][k]; in
    x's type unless ``dtype`` is given."""
    code, m, k, stride = _rows(x, "x")
    device = x.get_device()
    _check_integers(w, "w", k, device)
    out_code = code if dtype is None else _product_dtype(dtype)
    current = _stream(device)
    n = w.shape[0]
    out = x.new_empty((m, n)) if dtype is None else x.new_empty((m, n), dtype=dtype)
    size = _integer_room(m, n, k)
    room = _workspace(size, x)
    check(lib.smx_integer_linear(x.data_ptr(), stride, code, w.values.data_ptr(), w.scales.data_ptr(), m, n, k, out_code,
                                 out.data_ptr(), n, _at(room), size, current))
    return out


__all__ = ["BlockValues", "embed", "embed_gradient", "norm", "residual_norm", "residual_norm_gradient", "quantize",
           "block_product", "block_linear", "block_linear_gradient", "RowGroups", "group_rows", "grouped_linear",
           "grouped_linear_gradient", "gradient_norm", "clip_gradients", "IntegerValues", "quantize_integers",
           "integer_product", "integer_linear"]
