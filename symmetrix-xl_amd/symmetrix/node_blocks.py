"""A learned head over an evaluator's atoms, built of the node operators.

``NodeBlocks`` gives per-atom energies from species and per-atom descriptors: the species embedding
and a linear of the descriptors start each atom's row, residual blocks update it (a norm, an 8-bit
product that gives the update and its gate side by side, and the gated residual with the
next norm), and a vector reads the energy out.  With ``by_species`` each species has block weights of its own.  It trains
like any torch module; ``serve()`` keeps the shared weights in 8-bit blocks, where a block is two launches, the norm handing its
8-bit rows to the product, or in 8-bit integers, which are finer for a normed row's values.
First derivatives only: a gradient formed with ``create_graph`` raises ``RuntimeError`` when it is differentiated.

    python -m symmetrix.node_blocks --steps 300 --by-species --clip 1.0

fits it to the per-atom energies of a MACE evaluator on displaced SrTiO3 cells (random-init
weights of the tiny shape) and reports the error on a cell that it has not seen, trained and served.
"""

from __future__ import annotations

import argparse
import functools
import math
import time

import torch

from . import node_ops as ops


class _Undifferentiated(torch.autograd.Function):
    """Gradients as they are, whose own derivatives are an error instead of missing."""

    @staticmethod
    def forward(ctx, anchor, *grads):
        return tuple(g if g is None else g.clone() for g in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("symmetrix.node_blocks has first derivatives only: its gradients cannot be differentiated")


def _once(backward):
    """For a backward that records nothing: what it returns under ``create_graph`` raises when it is differentiated,
    whether or not the gradients that came in ask for a graph (the result depends on saved inputs as well)."""
    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        return _Undifferentiated.apply(torch.zeros((), requires_grad=True), *out)
    return wrapped


class _Embed(torch.autograd.Function):
    """Rows in the table's type, and the table's gradient summed in FP32 and rounded to it once."""

    @staticmethod
    def forward(ctx, table, types, scale):
        ctx.save_for_backward(types)
        ctx.num_types, ctx.scale = table.shape[0], scale
        return ops.embed(types, table, scale)

    @staticmethod
    @_once
    def backward(ctx, grad):
        types, = ctx.saved_tensors
        return ops.embed_gradient(types, grad.contiguous(), ctx.num_types, ctx.scale), None, None


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return ops.norm(x, weight, eps)

    @staticmethod
    @_once
    def backward(ctx, grad):
        x, weight = ctx.saved_tensors
        dx, *_, dw = ops.residual_norm_gradient(x, None, None, None, None, weight, None, grad.contiguous(), ctx.eps)
        return dx, dw, None


class _GatedResidual(torch.autograd.Function):
    """(y, h) from x and a block's output rows [update | gate logits].  These come in the rows' type: rounded to 16 bits in a
    16-bit head, which halves the largest array that a block writes and reads, at the size of the rounding of y itself."""

    @staticmethod
    def forward(ctx, x, both, post, scale, next_weight, eps):
        ctx.save_for_backward(x, both, post, scale, next_weight)
        ctx.eps = eps
        c = x.shape[1]
        return ops.residual_norm(x, both[:, :c], post, both[:, c:], scale, next_weight, eps)

    @staticmethod
    @_once
    def backward(ctx, grad_y, grad_h):
        x, both, post, scale, next_weight = ctx.saved_tensors
        c = x.shape[1]
        dx, dd, dg, dpost, dscale, dnext = ops.residual_norm_gradient(
            x, both[:, :c], post, both[:, c:], scale, next_weight, grad_y.contiguous(), grad_h.contiguous(), ctx.eps)
        return dx, torch.cat((dd, dg), 1), dpost, dscale, dnext, None


class _Linear(torch.autograd.Function):
    """x @ weight.T in 8-bit blocks, its gradients likewise; the weights are brought to x's type and then to blocks along
    both axes in one reading of them.  The weights' gradient is in their own type, whatever the rows' is."""

    @staticmethod
    def forward(ctx, x, weight):
        rows, ctx.w_columns = ops.quantize(weight.to(x.dtype), columns=True)
        y, ctx.x_columns = ops.block_linear(x, rows, keep=True)
        ctx.weight_dtype = weight.dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, grad):
        need_x, need_w = ctx.needs_input_grad
        dx, dw = ops.block_linear_gradient(grad.contiguous(), ctx.w_columns if need_x else None,
                                           ctx.x_columns if need_w else None, ctx.weight_dtype)
        return dx, dw


class _SpeciesLinear(torch.autograd.Function):
    """Each row through its species' matrix of weight [species][outputs][inputs], brought to x's type; FP32 sums, the weights'
    gradient in their own type."""

    @staticmethod
    def forward(ctx, x, weight, groups):
        w = weight.to(x.dtype)
        ctx.save_for_backward(x, w)
        ctx.groups, ctx.weight_dtype = groups, weight.dtype
        return ops.grouped_linear(x, w, groups)

    @staticmethod
    @_once
    def backward(ctx, grad):
        x, w = ctx.saved_tensors
        need_x, need_w, _ = ctx.needs_input_grad
        same = ctx.weight_dtype if ctx.weight_dtype is x.dtype else torch.float32
        dx, dw = ops.grouped_linear_gradient(grad.contiguous(), x if need_w else None, w if need_x else None, ctx.groups, same)
        return dx, None if dw is None else dw.to(ctx.weight_dtype), None


def _masked(types, descriptors, num_types):
    """(which atoms have a type of the table, the descriptors with zeros for the others): a masked atom's row is
    then zero all through, and shares no scale of 8-bit blocks with its neighbours."""
    there = (types >= 0) & (types < num_types)
    return there, torch.where(there[:, None], descriptors, 0)


def _energies(h, readout, shift, types, there):
    return torch.where(there, h.float() @ readout + shift[torch.where(there, types, 0).long()], 0)


class NodeBlocks(torch.nn.Module):
    """Per-atom energies of ``types`` [atoms] and ``descriptors`` [atoms][descriptors].  Rows are
    ``dtype``; parameters are float32.  With ``by_species`` a block's weights are a matrix for each type (up to 4,096 types).
    An atom whose type is outside [0, num_types) is masked, as in ``node_ops.embed``: its energy is zero, its descriptors are
    not looked at and nothing is learned from it."""

    def __init__(self, num_types, num_descriptors, channels=128, blocks=2, dtype=torch.float32, eps=1e-6, by_species=False):
        super().__init__()

        def normal(*shape, scale=1.0):
            return torch.nn.Parameter(scale * torch.randn(*shape))

        def ones(value=1.0):
            return torch.nn.Parameter(torch.full((channels,), value))
        self.dtype, self.eps, self.channels, self.by_species = dtype, eps, channels, by_species
        own = (num_types,) if by_species else ()
        self.table = normal(num_types, channels, scale=1 / math.sqrt(channels))
        self.lift = normal(channels, num_descriptors, scale=1 / math.sqrt(num_descriptors))
        self.before = ones()
        self.weights = torch.nn.ParameterList(
            [normal(*own, 2 * channels, channels, scale=1 / math.sqrt(channels)) for _ in range(blocks)])
        self.post = torch.nn.ParameterList([ones() for _ in range(blocks)])
        self.scale = torch.nn.ParameterList([ones(0.5) for _ in range(blocks)])
        self.next = torch.nn.ParameterList([ones() for _ in range(blocks)])
        self.readout = normal(channels, scale=0.1 / math.sqrt(channels))
        self.shift = torch.nn.Parameter(torch.zeros(num_types))

    def forward(self, types, descriptors):
        t = self.dtype
        there, descriptors = _masked(types, descriptors, self.table.shape[0])
        x = _Embed.apply(self.table.to(t), types, math.sqrt(self.channels))
        x = x + _Linear.apply(descriptors.to(t), self.lift)
        h = _Norm.apply(x, self.before, self.eps)
        groups = ops.group_rows(types, self.table.shape[0]) if self.by_species else None
        for w, post, scale, nxt in zip(self.weights, self.post, self.scale, self.next):
            both = _SpeciesLinear.apply(h, w, groups) if self.by_species else _Linear.apply(h, w)
            x, h = _GatedResidual.apply(x, both, post, scale, nxt, self.eps)
        return _energies(h, self.readout, self.shift, types, there)

    def serve(self, form="blocks"):
        """A function of (types, descriptors) with the present weights in 8-bit ``form``: "blocks" (E4M3 with a scale for each
        128) or "integers" (with a scale for each row).  Weights by species are kept in the rows' type."""
        if form not in ("blocks", "integers"):
            raise ValueError("weights are served in blocks or integers")
        quantize, linear = (ops.quantize, ops.block_linear) if form == "blocks" else (ops.quantize_integers, ops.integer_linear)
        by_species, handed = self.by_species, form == "blocks" and not self.by_species
        with torch.no_grad():
            t = self.dtype
            table, lift = self.table.detach().to(t).clone(), quantize(self.lift.detach().to(t))
            weights = [w.detach().to(t).clone() if by_species else quantize(w.detach().to(t)) for w in self.weights]
            before, readout, shift = (p.detach().clone() for p in (self.before, self.readout, self.shift))
            vectors = [tuple(p.detach().clone() for p in v) for v in zip(self.post, self.scale, self.next)]
        c, eps = self.channels, self.eps

        @torch.no_grad()
        def energies(types, descriptors):
            there, descriptors = _masked(types, descriptors, table.shape[0])
            x = ops.embed(types, table, math.sqrt(c))
            x += linear(descriptors.to(t), lift)
            # (rows handed to a block product are in blocks already)
            h = ops.norm(x, before, eps, quantized=handed)
            groups = ops.group_rows(types, table.shape[0]) if by_species and weights else None
            for k, (w, (post, scale, nxt)) in enumerate(zip(weights, vectors)):
                if by_species:
                    both = ops.grouped_linear(h, w, groups)
                else:
                    both = ops.block_product(h, w, t) if handed else ops.integer_linear(h, w)
                x, h = ops.residual_norm(x, both[:, :c], post, both[:, c:], scale, nxt, eps,
                                         quantized=handed and k + 1 < len(weights))
            return _energies(h if weights else ops.norm(x, before, eps), readout, shift, types, there)
        return energies


# ---- the example ----


def descriptors_of(system, type_of, cutoff=5.0, radial=8):
    """Sums over each atom's neighbours, by their species, of Gaussians of the distance under a
    smooth cutoff: [atoms][species x radial] float32."""
    import numpy as np

    from .neighbors import neighbor_list_ijS
    i, j, s = neighbor_list_ijS(system["positions"], system["cell"], system["pbc"], cutoff)
    d = np.linalg.norm(system["positions"][j] - system["positions"][i] + s @ system["cell"], axis=1)
    centres = np.linspace(1.5, cutoff, radial)
    g = np.exp(-((d[:, None] - centres) / 0.4) ** 2) * (0.5 + 0.5 * np.cos(math.pi * d / cutoff))[:, None]
    n = len(system["numbers"])
    out = np.zeros((n, len(type_of), radial))
    np.add.at(out, (i, np.vectorize(type_of.get)(system["numbers"][j])), g)
    return out.reshape(n, -1).astype(np.float32)


def fit(steps=300, cells=3, channels=128, blocks=2, dtype=torch.float32, seed=0, report=print, by_species=False, clip=None,
        form="blocks"):
    """Fits the head to an evaluator's per-atom energies; the errors (eV/atom, root mean square) on an unseen cell of
    the trained head and of the served one, and that of the species' means.  ``clip``: the largest norm of a step's gradients."""
    import numpy as np

    from . import random_model, systems
    from .mace_kokkos import MACEKokkosFloat
    torch.manual_seed(seed)
    ev = MACEKokkosFloat(random_model.cached_model("tiny"))
    type_of = {z: k for k, z in enumerate(ev.atomic_numbers)}
    data = []
    for k in range(5):  # the last is the unseen one
        system = systems.srtio3_supercell(cells, sigma=0.1, seed=seed + k)
        types = np.vectorize(type_of.get)(system["numbers"]).astype(np.int32)
        cell = system["cell"]
        g = ev._prepare_periodic_factorized_graph(types, system["positions"].ravel(), cell.ravel(),
                                                  np.linalg.inv(cell).ravel(), ev.r_cut + 0.5)
        ev._compute_prepared_factorized_positions(g["generation"], system["positions"].ravel())
        data.append((types, descriptors_of(system, type_of), np.array(ev.node_energies)))
    types, desc, energy = (torch.from_numpy(np.concatenate([d[n] for d in data])).cuda() for n in range(3))
    n = len(data[0][0])
    train, test = slice(0, 4 * n), slice(4 * n, 5 * n)
    means = torch.stack([energy[train][types[train] == k].mean() for k in range(len(type_of))])
    desc = (desc - desc[train].mean(0)) / (desc[train].std(0) + 1e-6)
    target = energy - means[types.long()]
    unit = target[train].std()
    target = (target / unit).float()
    model = NodeBlocks(len(type_of), desc.shape[1], channels, blocks, dtype, by_species=by_species).cuda()
    adam = torch.optim.Adam(model.parameters(), lr=2e-3)
    begin = time.perf_counter()
    for step in range(steps):
        adam.zero_grad(set_to_none=True)
        loss = (model(types[train], desc[train]) - target[train]).square().mean()
        loss.backward()
        if clip is not None:
            ops.clip_gradients([p.grad for p in model.parameters()], clip)
        adam.step()
        if report and (step % 100 == 0 or step + 1 == steps):
            report("step %d: loss %.4f" % (step, loss.item()))
    took = time.perf_counter() - begin

    def error(values):
        return float(((values - target[test]) * unit).square().mean().sqrt())
    with torch.no_grad():
        trained, served = error(model(types[test], desc[test])), error(model.serve(form)(types[test], desc[test]))
    result = {"trained": trained, "served": served, "means": error(torch.zeros_like(target[test])),
              "ms_per_step": 1e3 * took / max(1, steps)}
    if report:
        report("unseen cell, eV/atom: %.2e trained, %.2e served, %.2e from the species' means; %.2f ms a step"
               % (trained, served, result["means"], result["ms_per_step"]))
    return result


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--cells", type=int, default=3)
    ap.add_argument("--channels", type=int, default=128)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--dtype", choices=("float32", "bfloat16", "float16"), default="float32")
    ap.add_argument("--by-species", action="store_true", help="block weights for each species")
    ap.add_argument("--clip", type=float, help="the largest norm of a step's gradients")
    ap.add_argument("--form", choices=("blocks", "integers"), default="blocks", help="the served weights' 8-bit form")
    args = ap.parse_args(argv)
    fit(args.steps, args.cells, args.channels, args.blocks, getattr(torch, args.dtype), by_species=args.by_species,
        clip=args.clip, form=args.form)


if __name__ == "__main__":
    main()
