"""The operators that symmetrix.node_blocks is built of, in plain torch on any device and without 8-bit rounding, so that
its autograd functions and the head around them can be run on the CPU."""

import torch


def embed(types, table, scale=1.0):
    there = (types >= 0) & (types < table.shape[0])
    return torch.where(there[:, None], table[torch.where(there, types, 0).long()] * scale, 0.0)


def embed_gradient(types, grad, num_types, scale=1.0):
    there = (types >= 0) & (types < num_types)
    out = torch.zeros(num_types, grad.shape[1], dtype=grad.dtype)
    return out.index_add_(0, types[there].long(), grad[there]) * scale


def _unit(x, eps):
    return x / torch.sqrt(x.square().mean(1, keepdim=True) + eps)


def norm(x, weight, eps=1e-6, quantized=False):
    return (weight * _unit(x.float(), eps)).to(x.dtype)


def residual_norm(x, d, post, gate=None, scale=None, next_weight=None, eps=1e-6, quantized=False):
    gate = 1 if gate is None else torch.sigmoid(gate.float())
    y = x.float() + (1 if scale is None else scale) * gate * post * _unit(d.float(), eps)
    return y.to(x.dtype), None if next_weight is None else norm(y, next_weight, eps).to(x.dtype)


def residual_norm_gradient(x, d, post, gate, scale, next_weight, grad_y, grad_h, eps=1e-6):
    given = (x, d, gate, post, scale, next_weight)
    leaves = [None if t is None else t.detach().requires_grad_() for t in given]
    x, d, gate, post, scale, next_weight = leaves
    with torch.enable_grad():
        y, h = (x, norm(x, next_weight, eps)) if d is None else residual_norm(x, d, post, gate, scale, next_weight, eps)
        loss = sum((a * b).sum() for a, b in ((y, grad_y), (h, grad_h)) if b is not None)
        got = iter(torch.autograd.grad(loss, [t for t in leaves if t is not None]))
    return tuple(None if t is None else next(got) for t in leaves)


def quantize(x, rows=True, columns=False):
    a, b = x.clone(), x.T.clone()
    return (a, b) if rows and columns else a if rows else b


def block_product(a, b, dtype=torch.float32):
    return (a.float() @ b.float().T).to(dtype)


def block_linear(x, w, dtype=None, keep=False):
    y = block_product(x, w, x.dtype if dtype is None else dtype)
    return (y, x.T.clone()) if keep else y


def block_linear_gradient(grad, w_columns, x_columns, dtype=None):
    return (None if w_columns is None else block_product(grad, w_columns, grad.dtype),
            None if x_columns is None else block_product(grad.T, x_columns, dtype or torch.float32))
