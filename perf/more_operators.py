"""Performance cases of the node operators for rows by kind and for integers: the
grouping of rows by their kind, products with a weight matrix for each kind and their
gradients, the norm of many gradients with clipping, and products in 8-bit integers with
scales for each row.

With ``own`` false a case is computed in plain torch operations in 32 bits, exact integer
sums and the norm of many values in 64; with ``own`` true by the calls of
``symmetrix.node_ops``.  ``exact`` is the same quantity from its definition in float64.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
MAX_NORM = 1.0


def listed():
    return [
        # the species of a unit-test cell: latency is all of it
        {"name": "groups-135", "kind": "groups", "rows": 135, "types": 89, "index": "i32", "spread": "crystal"},
        # many kinds with a long tail (environment types) in one training batch, some rows masked out
        {"name": "groups-131071", "kind": "groups", "rows": 131071, "types": 1009, "index": "i64", "spread": "tail"},
        # one served row through the weights of its kind: these bytes are all of it
        {"name": "grouped-1x2048x4096", "kind": "grouped", "direction": "forward", "rows": 1, "types": 64,
         "inputs": 2048, "outputs": 4096, "dtype": "bf16", "spread": "even"},
        # a small served batch, a few rows of each kind
        {"name": "grouped-147x1024x2048", "kind": "grouped", "direction": "forward", "rows": 147, "types": 32,
         "inputs": 1024, "outputs": 2048, "dtype": "f16", "spread": "even"},
        # the wide water box of the benchmark, two species, a training step in FP32
        {"name": "grouped-train-water-30000x256x512", "kind": "grouped", "direction": "train", "rows": 30000, "types": 2,
         "inputs": 256, "outputs": 512, "dtype": "f32", "spread": "crystal"},
        # an odd count of atoms of the 89-element table, an odd width, most kinds rare and some rows masked out
        {"name": "grouped-train-6791x224x999", "kind": "grouped", "direction": "train", "rows": 6791, "types": 89,
         "inputs": 224, "outputs": 999, "dtype": "f16", "spread": "tail"},
        # the ten species of the irregular 20,000-atom box through one block's weights, a training step
        {"name": "grouped-train-20000x512x1024", "kind": "grouped", "direction": "train", "rows": 20000, "types": 10,
         "inputs": 512, "outputs": 1024, "dtype": "bf16", "spread": "even"},
        # the largest: a long batch over many kinds
        {"name": "grouped-32768x2048x4096", "kind": "grouped", "direction": "forward", "rows": 32768, "types": 64,
         "inputs": 2048, "outputs": 4096, "dtype": "bf16", "spread": "even"},
        # the gradients of a small head: one launch is most of it
        {"name": "clip-head-14", "kind": "clip", "direction": "clip", "tensors": 14, "values": 84099, "dtype": "f32",
         "out": "f32"},
        # the gradients of a large model in 16 bits, brought to FP32 for the optimiser
        {"name": "clip-120-402M", "kind": "clip", "direction": "clip", "tensors": 120, "values": 402000001,
         "dtype": "bf16", "out": "f32"},
        # the product of one served row: the weights' bytes are all of it
        {"name": "integers-1x4096x8192", "kind": "integers", "direction": "linear", "rows": 1, "inputs": 4096,
         "outputs": 8192, "dtype": "bf16"},
        # the largest product
        {"name": "integers-16384x8192x8192", "kind": "integers", "direction": "linear", "rows": 16384, "inputs": 8192,
         "outputs": 8192, "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm; odd half of the time."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        n |= 1
    return max(lo, min(hi, n))


def draw(rng):
    kind = rng.choice(["groups", "grouped", "grouped", "grouped", "clip", "integers", "integers"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    spread = rng.choice(["crystal", "even", "tail"])
    if kind == "groups":
        return {"kind": kind, "rows": _spread(rng, 1, 300000), "types": _spread(rng, 1, 4096),
                "index": rng.choice(["i32", "i64"]), "spread": spread}
    if kind == "grouped":
        train = rng.random() < 0.5
        k, n = _spread(rng, 16, 4096), _spread(rng, 16, 4096)
        types = max(1, min(_spread(rng, 1, 512), (1 << 28) // (k * n)))
        rows = max(1, min(_spread(rng, 1, 32768), (1 << (35 if dtype == "f32" else 36 if train else 38)) // (k * n)))
        return {"kind": kind, "direction": "train" if train else "forward", "rows": rows, "types": types, "inputs": k,
                "outputs": n, "dtype": dtype, "spread": spread}
    if kind == "clip":
        tensors = _spread(rng, 1, 1000)
        return {"kind": kind, "direction": rng.choice(["clip", "clip", "norm"]), "tensors": tensors,
                "values": max(tensors, _spread(rng, 1000, 300000000)), "dtype": dtype,
                "out": rng.choice([dtype, "f32"])}
    k, n = _spread(rng, 32, 8192), _spread(rng, 32, 8192)
    direction = rng.choice(["linear", "linear", "quantize"])
    return {"kind": kind, "direction": direction, "rows": _spread(rng, 1, 16384), "inputs": k,
            "outputs": n if direction == "linear" else 0, "dtype": dtype}


def _ops():
    at = os.path.join(os.getcwd(), "symmetrix-xl_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from symmetrix import node_ops
    return node_ops


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale).to(dtype)


def _rows(gen, rows, channels, dtype):
    """Activations: rows of unequal size, and a few channels that stand out."""
    x = torch.randn((rows, channels), generator=gen, device=gen.device)
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device=gen.device))
    x *= 1 + 7 * (torch.rand((1, channels), generator=gen, device=gen.device) < 0.02)
    return x.to(dtype)


def _types(gen, case):
    t, v, device = case["rows"], case["types"], gen.device
    if case["spread"] == "crystal":  # a few species of the table, shuffled atoms
        few = torch.randint(0, v, (min(v, 5),), generator=gen, device=device)
        few[0] = v - 1
        few[-1] = 0
        z = few[torch.randint(0, few.numel(), (t,), generator=gen, device=device)]
    elif case["spread"] == "even":
        z = torch.randint(0, v, (t,), generator=gen, device=device)
    else:  # frequent kinds and a long tail, 2% of the rows masked out
        u = torch.rand(t, generator=gen, device=device)
        z = (torch.pow(float(v), u) - 1).long().clamp(0, v - 1)
        z = (z * 7919 + 13) % v
        z = torch.where(torch.rand(t, generator=gen, device=device) < 0.02, -1, z)
    return z


def _sizes(case):
    """The values of each tensor: vectors, tables and matrices of a model, of very unequal sizes."""
    rng = random.Random(case["tensors"])
    share = [math.exp(rng.uniform(0, 7)) for _ in range(case["tensors"])]
    spare = case["values"] - case["tensors"]
    sizes = [1 + int(spare * s / sum(share)) for s in share]
    sizes[-1] += case["values"] - sum(sizes)
    return sizes


def prepare(case, seed):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=device)
    gen.manual_seed(int(seed))
    s = {"case": case}
    kind = case["kind"]
    if kind == "groups":
        s["types"] = _types(gen, case).to(torch.int64 if case["index"] == "i64" else torch.int32)
        return s
    dtype = DTYPES[case["dtype"]]
    if kind == "grouped":
        t, v, k, n = case["rows"], case["types"], case["inputs"], case["outputs"]
        z = _types(gen, case)
        # made once for a batch and used by every block and direction
        if own:
            s["groups"] = _ops().group_rows(z, v)
        else:
            s["members"] = [(g, torch.nonzero(z == g)[:, 0]) for g in torch.unique(z).tolist() if g >= 0]
        s["x"] = _rows(gen, t, k, dtype)
        s["w"] = _normal(gen, (v, n, k), dtype, 1 / math.sqrt(k))
        if case["direction"] == "train":
            s["grad"] = _normal(gen, (t, n), dtype)
        s["types"] = z
    elif kind == "clip":
        # FP16 gradients come with the loss scaled up
        s["scale"] = 1 / 1024 if case["dtype"] == "f16" else 1.0
        unit = 1 / (s["scale"] * math.sqrt(case["values"]))
        s["grads"] = [_normal(gen, (n,), dtype, unit * math.exp(0.5 + 0.1 * (i % 7))) for i, n in
                      enumerate(_sizes(case))]
        if case["direction"] == "clip":  # one buffer of all gradients, as an optimiser keeps it
            s["flat"] = torch.empty(case["values"], dtype=DTYPES[case["out"]], device=device)
            s["out"] = list(torch.split(s["flat"], _sizes(case)))
    else:
        s["x"] = _rows(gen, case["rows"], case["inputs"], dtype)
        if case["direction"] == "linear":
            w = _normal(gen, (case["outputs"], case["inputs"]), dtype, 1 / math.sqrt(case["inputs"]))
            s["w"] = _ops().quantize_integers(w) if own else _integers(w)
    return s


# ---- the plain form ----


def _integers(x):
    """(whole numbers up to 127 in magnitude, the FP32 scale of each row)"""
    x = x.float()
    scale = (x.abs().amax(1, keepdim=True) / 127).clamp(min=2.0 ** -126)
    # the quotient in 64 bits: in 32 it may round onto a border that it is not on
    return (x.double() / scale.double()).round().to(torch.int8), scale


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "groups":
        v, z = case["types"], s["types"]
        key = torch.where((z >= 0) & (z < v), z, v).long()
        order = torch.sort(key, stable=True).indices
        counts = torch.zeros(v + 1, dtype=torch.int64, device=z.device).index_add_(0, key, torch.ones_like(key))
        offsets = torch.nn.functional.pad(torch.cumsum(counts[:-1], 0), (1, 0))
        return [order.to(torch.int32), offsets.to(torch.int32)]
    dtype = DTYPES[case["dtype"]]
    if kind == "grouped":
        x, w = s["x"], s["w"]
        y = torch.zeros((case["rows"], case["outputs"]), device=x.device)
        if case["direction"] == "forward":
            for g, at in s["members"]:
                y[at] = x[at].float() @ w[g].float().T
            return y.to(dtype)
        grad, dx = s["grad"], torch.zeros(x.shape, device=x.device)
        dw = torch.zeros(w.shape, device=x.device)
        for g, at in s["members"]:
            xg, wg, gg = x[at].float(), w[g].float(), grad[at].float()
            y[at] = xg @ wg.T
            dx[at] = gg @ wg
            dw[g] = gg.T @ xg
        return [y.to(dtype), dx.to(dtype), dw]
    if kind == "clip":
        # (squares and their sum in 64 bits: hundreds of millions of values)
        total = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt() * s["scale"]
        if case["direction"] == "norm":
            return total.float()
        factor = ((MAX_NORM / total).clamp(max=1.0) * s["scale"]).float()
        for g, o in zip(s["grads"], s["out"]):
            o.copy_(g.float() * factor)
        return [total.float(), s["flat"]]
    q, scale = _integers(s["x"])
    if case["direction"] == "quantize":
        return q.float() * scale
    # (64-bit sums of whole numbers are exact, 32-bit ones are not)
    wq, ws = s["w"]
    return ((q.double() @ wq.double().T).float() * scale * ws.T).to(dtype)


# ---- the framework's calls ----


def _own(s):
    ops, case = _ops(), s["case"]
    kind = case["kind"]
    if kind == "groups":
        groups = ops.group_rows(s["types"], case["types"])
        return [groups.order, groups.offsets]
    if kind == "grouped":
        y = ops.grouped_linear(s["x"], s["w"], s["groups"])
        if case["direction"] == "forward":
            return y
        return [y, *ops.grouped_linear_gradient(s["grad"], s["x"], s["w"], s["groups"])]
    if kind == "clip":
        if case["direction"] == "norm":
            return ops.gradient_norm(s["grads"], scale=s["scale"])
        return [ops.clip_gradients(s["grads"], MAX_NORM, scale=s["scale"], out=s["out"]), s["flat"]]
    if case["direction"] == "quantize":
        return ops.quantize_integers(s["x"]).float()
    return ops.integer_linear(s["x"], s["w"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    kind = case["kind"]
    if kind == "groups":
        return {"bytes": case["rows"] * (4 + (8 if case["index"] == "i64" else 4)) + 4 * (case["types"] + 1),
                "flops": case["rows"]}
    e = SIZES[case["dtype"]]
    if kind == "grouped":
        t, v, k, n = case["rows"], case["types"], case["inputs"], case["outputs"]
        # the weights of kinds that have rows
        present = min(v, 5) if case["spread"] == "crystal" else v
        read = min(present, t) * n * k
        if case["direction"] == "forward":
            return {"bytes": e * (t * (k + n) + read), "flops": 2 * t * k * n}
        return {"bytes": e * (2 * t * (k + n) + read) + 4 * v * n * k, "flops": 6 * t * k * n}
    if kind == "clip":
        wrote = SIZES[case["out"]] if case["direction"] == "clip" else 0
        return {"bytes": case["values"] * (e + wrote), "flops": case["values"] * (3 if wrote else 2)}
    t, k, n = case["rows"], case["inputs"], case["outputs"]
    if case["direction"] == "quantize":
        return {"bytes": t * k * (e + 4), "flops": 3 * t * k}
    return {"bytes": e * t * (k + n) + n * k + 4 * n, "flops": 2 * t * k * n}


# ---- float64, from the definitions ----


def _rounded(x):
    """x in float64 as the multiples of its rows' scales that stand for it: a scale is the FP32
    number nearest to a 127th of the row's largest magnitude, or 2^-126."""
    x = x.double()
    scale = (x.abs().max(1, keepdim=True).values / 127).float().double()
    scale = torch.maximum(scale, torch.full_like(scale, 2.0 ** -126))
    return torch.round(x / scale) * scale


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "groups":
        z, v = s["types"].cpu().numpy().astype(np.int64), case["types"]
        z[(z < 0) | (z >= v)] = v
        order = np.argsort(z, kind="stable")
        offsets = np.searchsorted(z[order], np.arange(v + 1))
        return [torch.from_numpy(a.astype(np.int32)) for a in (order, offsets)]
    if kind == "grouped":
        z, train = s["types"], case["direction"] == "train"
        t, k = s["x"].shape
        y = torch.zeros((t, case["outputs"]), dtype=torch.float64, device=z.device)
        dx = torch.zeros((t, k), dtype=torch.float64, device=z.device)
        dw = []
        for g in range(case["types"]):
            at = z == g
            x, w = s["x"][at].double(), s["w"][g].double()
            y[at] = torch.matmul(x, w.mT.contiguous())
            if train:
                grad = s["grad"][at].double()
                dx[at] = torch.matmul(grad, w)
                dw.append(torch.matmul(grad.mT.contiguous(), x).float())
        return [y, dx, torch.stack(dw)] if train else y
    if kind == "clip":
        total = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in s["grads"])) * s["scale"]
        norm = torch.tensor(total, dtype=torch.float64)
        if case["direction"] == "norm":
            return norm
        factor = s["scale"] * (MAX_NORM / total if total > MAX_NORM else 1.0)
        return [norm, torch.cat(s["grads"]).double() * factor]
    x = _rounded(s["x"])
    if case["direction"] == "quantize":
        return x
    q, scale = s["w"]
    return x @ (q.double() * scale.double()).T.contiguous()
