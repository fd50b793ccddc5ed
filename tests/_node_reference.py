"""The node operators' definitions in float64 on the CPU, with bounds of what FP32
sums and one rounding to the outputs' type may add to them."""

import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# a value below the type's least normal is off by half of its least subnormal
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def d(t):
    return None if t is None else t.detach().cpu().double()


def assert_within(got, want, bound, dtype=None):
    """|got - want| <= bound + the rounding of want to got's type, NaN in the same places, and an infinity
    where want is beyond the type."""
    dtype = dtype or got.dtype
    got = d(got)
    want = torch.where(want.abs() > torch.finfo(dtype).max, torch.sign(want) * math.inf, want)
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and (got * want)[torch.isinf(want)].ge(0).all()
    fine = torch.isfinite(want)
    off = (got - want).abs()[fine]
    limit = (torch.as_tensor(bound).expand_as(want) + 1.0001 * UNIT[dtype] * want.abs() + LEAST[dtype])[fine]
    worst = (off / limit).max().item() if off.numel() else 0.0
    assert worst <= 1.0, "off by %.3g of the bound" % worst


# ---- 8-bit blocks ----


def quantized(x):
    """(values that the blocks stand for, scale bytes) of x [r][k]; NaN and infinities as NaN."""
    x = d(x)
    r, k = x.shape
    blocks = -(-k // 128)
    x = torch.cat([x, x.new_zeros(r, blocks * 128 - k)], 1).reshape(r, blocks, 128)
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), 0.0).amax(2)
    byte = torch.zeros(r, blocks, dtype=torch.int64)
    for i in range(r):
        for b in range(blocks):
            m, e = math.frexp(top[i, b].item())  # m in [0.5, 1): top = 2m 2^(e-1), and 448 = 1.75 * 2^8
            byte[i, b] = 0 if m == 0 else max(0, e - 9 + (1 if m > 0.875 else 0) + 127)
    scale = torch.exp2((byte - 127).double())[:, :, None]
    v = torch.where(finite, x, 0.0) / scale
    grid = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    q = torch.round(v / grid) * grid
    q = torch.where(finite, q * scale, math.nan)
    return q.reshape(r, blocks * 128)[:, :k], byte


def product(a, b, extra=0):
    """a @ b.T and the bound of FP32 sums of its terms."""
    want = a @ b.T
    bound = (a.shape[1] + 8 + extra) * 2.0 ** -23 * (a.abs() @ b.abs().T)
    return want, bound


# ---- residual norm ----


class Norm:
    """Forward and backward of the residual norm with bounds: each quantity's magnitude is the sum of
    its terms' magnitudes, and FP32 arithmetic adds at most (channels + 64) 2^-23 of it (sums of
    `channels` terms, the reciprocal square root, the sigmoid's exponential and a few products)."""

    def __init__(self, x, dd, post, gate, scale, nxt, eps):
        self.x, self.d = d(x), d(dd)
        r, c = self.x.shape
        self.rel = (c + 64) * 2.0 ** -23
        one = torch.ones(1, dtype=torch.float64)
        self.post, self.scale = (d(post) if post is not None else one), (d(scale) if scale is not None else one)
        self.next = d(nxt)
        self.gate = d(gate)
        if self.d is not None:
            self.s = torch.sigmoid(self.gate) if gate is not None else one
            # the sigmoid's argument enters its exponential: |g| more roundings
            self.rel = self.rel + (self.gate.abs().max().item() if gate is not None and self.gate.numel() else 0) * 2.0 ** -23
            self.r1 = 1 / torch.sqrt(self.d.pow(2).mean(1, keepdim=True) + eps)
            self.u = self.d * self.r1
            self.n = self.u * self.post
            step = self.scale * self.s * self.n
        else:
            step = torch.zeros_like(self.x)
        self.y = self.x + step
        self.y_bound = self.rel * step.abs() + 2.0 ** -23 * self.y.abs()
        self.r2 = 1 / torch.sqrt(self.y.pow(2).mean(1, keepdim=True) + eps)
        self.v = self.y * self.r2
        # h moves with y's own error and, through the norm, with the error's share of the row
        share = self.y_bound.norm(dim=1, keepdim=True) / self.y.norm(dim=1, keepdim=True).clamp(min=1e-30)
        self.v_bound = self.r2 * self.y_bound + (self.rel + share) * self.v.abs()
        if self.next is not None:
            self.h = self.v * self.next
            self.h_bound = self.v_bound * self.next.abs() + self.rel * self.h.abs()

    def backward(self, gy, gh):
        rel = 2 * self.rel
        c = self.x.shape[1]
        zero = torch.zeros_like(self.x)
        gy = zero if gy is None else d(gy)
        out, bound = {}, {}
        dx, mag, more = gy, gy.abs(), zero
        if gh is not None:
            gh = d(gh)
            q = gh * self.next
            m = (q * self.v).mean(1, keepdim=True)
            dx = gy + self.r2 * (q - self.v * m)
            mag = gy.abs() + self.r2 * (q.abs() + self.v.abs() * (q * self.v).abs().mean(1, keepdim=True))
            # what v's own error does
            more = self.r2 * (self.v_bound * (q * self.v).abs().mean(1, keepdim=True) +
                              self.v.abs() * (q.abs() * self.v_bound).mean(1, keepdim=True))
            out["next"] = (gh * self.v).sum(0)
            bound["next"] = (gh.abs() * self.v_bound).sum(0) + (rel + self.x.shape[0] * 2.0 ** -23) * (gh * self.v).abs().sum(0)
        elif self.next is not None:
            out["next"], bound["next"] = zero.sum(0), zero.sum(0)
        out["x"] = dx
        ex = rel * mag + more
        bound["x"] = ex
        if self.d is None:
            return out, bound
        p, pm = dx * self.scale * self.s, mag * (self.scale * self.s).abs()
        t, tm = p * self.post, pm * self.post.abs()
        et = ex * (self.scale * self.s * self.post).abs() + rel * tm
        out["d"] = self.r1 * (t - self.u * (t * self.u).mean(1, keepdim=True))
        bound["d"] = self.r1 * (et + self.u.abs() * (et * self.u.abs()).mean(1, keepdim=True)) + \
            rel * self.r1 * (tm + self.u.abs() * (tm * self.u.abs()).mean(1, keepdim=True))
        rows = self.x.shape[0] * 2.0 ** -23 + rel
        out["post"] = (p * self.u).sum(0)
        bound["post"] = rows * (pm * self.u.abs()).sum(0) + (ex * (self.scale * self.s * self.u).abs()).sum(0)
        out["scale"] = (dx * self.s * self.n).sum(0)
        bound["scale"] = rows * (mag * (self.s * self.n).abs()).sum(0) + (ex * (self.s * self.n).abs()).sum(0)
        if self.gate is not None:
            # 1 - s from s: the difference is off by s's own rounding
            f = self.scale * self.n * self.s * (1 - self.s)
            fm = (self.scale * self.n).abs() * self.s
            g, eg = dx * f, ex * f.abs() + rel * mag * fm
            if self.gate.dim() == 1:
                g, eg = g.sum(0), eg.sum(0) + rows * (mag * fm).sum(0)
            elif self.gate.shape[1] == 1 and c > 1:
                g, eg = g.sum(1, keepdim=True), eg.sum(1, keepdim=True) + rel * (mag * fm).sum(1, keepdim=True)
            out["gate"], bound["gate"] = g, eg
        return out, bound
