"""A deformable-attention encoder layer from this package's operators alone.

The layer of Deformable-DETR's encoder (and, with its own reference points, of
BEVFormer's): value, offset and weight projections, multi-scale deformable
attention, output projection onto the residual, norm, feed-forward onto the
residual, norm. Every product with its bias, activation and residual is one
``linear_act``; with ``checkpoint="int8"`` the feed-forward and the norms keep
their inputs for the backward pass in 8 bits.

In training with ``dropout``, the output of either block is dropped out, added to the
residual and normalised by one ``add_norm``, and the feed-forward's hidden rows go
through ``dropout``. ``gated`` takes the feed-forward's first product from
``gated_linear`` (dropout included); ``norms="branch"`` normalises what a block adds
instead of the sum, with a gate per channel (``norm_add``).

    python -m muspace_b200.encoder                  # a training step, timed, with and without checkpoints
    python -m muspace_b200.encoder --queries 900 --forward
    python -m muspace_b200.encoder --dropout 0.1 --gated [--norms branch]
"""

from __future__ import annotations

import argparse

import torch
from torch import nn

from . import cases
from .ops import (
    add_norm, dropout as drop, gated_linear, layer_norm, linear_act, multi_scale_deformable_attn, norm_add)


class _Linear(nn.Module):
    def __init__(self, in_features: int, out_features: int, **kind):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(out_features, in_features, **kind))
        self.bias = nn.Parameter(torch.zeros(out_features, **kind))
        nn.init.xavier_uniform_(self.weight)

    def forward(self, x, residual=None, **how):
        return linear_act(x, self.weight, self.bias, residual, **how)


class _Norm(nn.Module):
    def __init__(self, width: int, gate: bool = False, **kind):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(width, **kind))
        self.bias = nn.Parameter(torch.zeros(width, **kind))
        self.gate = nn.Parameter(torch.ones(width, **kind)) if gate else None

    def forward(self, x, **how):
        return layer_norm(x, self.weight, self.bias, **how)

    def join(self, x, residual, **how):
        """A block's output onto the residual: the norm of the sum, or the sum with the gated norm of the output."""
        if self.gate is None:
            return add_norm(x, residual, self.weight, self.bias, **how)
        return norm_add(x, residual, self.weight, self.bias, gate=self.gate, **how)


class DeformableEncoderLayer(nn.Module):
    """Post-norm encoder layer; ``forward`` takes queries ``(B, Lq, C)``, the feature
    rows ``(B, Lin, C)`` that they sample (the queries themselves in an encoder),
    reference points ``(B, Lq, L, 2)`` as (x, y) in [0, 1] and the level tables of
    ``multi_scale_deformable_attn``.

    In training with ``dropout`` it needs a ``seed`` too, an integer or an int64 tensor on
    the device, another one for each step; ``index`` tells a model's layers apart."""

    def __init__(self, width: int = 256, hidden: int = 1024, heads: int = 8, levels: int = 4, points: int = 4,
                 activation: str = "relu", checkpoint: str | None = None, device=None, dtype=None, *,
                 dropout: float = 0.0, gated: bool = False, norms: str = "sum", index: int = 0):
        super().__init__()
        if width % heads:
            raise ValueError("width must be divisible by heads")
        if norms not in ("sum", "branch"):
            raise ValueError(f"norms must be 'sum' or 'branch', got {norms!r}")
        if checkpoint is not None and (dropout or gated or norms == "branch"):
            raise ValueError("checkpoints go with the plain layer: no dropout, gated product or norms of the branch")
        kind = {"device": device, "dtype": dtype}
        self.heads, self.levels, self.points = heads, levels, points
        self.activation, self.checkpoint = activation, checkpoint
        self.dropout, self.gated, self.branch, self.index = dropout, gated, norms == "branch", index
        self.value = _Linear(width, width, **kind)
        self.offsets = _Linear(width, heads * levels * points * 2, **kind)
        self.weights = _Linear(width, heads * levels * points, **kind)
        self.output = _Linear(width, width, **kind)
        self.up = _Linear(width, 2 * hidden if gated else hidden, **kind)
        self.down = _Linear(hidden, width, **kind)
        self.norm1 = _Norm(width, self.branch, **kind)
        self.norm2 = _Norm(width, self.branch, **kind)

    def forward(self, queries, features, reference_points, spatial_shapes, level_start_index, position=None, seed=None):
        batch, count, width = queries.shape
        placed = queries if position is None else queries + position
        value = self.value(features).view(batch, features.size(1), self.heads, width // self.heads)
        shape = (batch, count, self.heads, self.levels, self.points)
        offsets = self.offsets(placed).view(*shape, 2)
        weights = self.weights(placed).view(*shape[:3], -1).softmax(-1).view(shape)
        size = spatial_shapes.flip(-1).to(offsets.dtype)  # (W, H) of each level
        locations = reference_points[:, :, None, :, None, :] + offsets / size[None, None, None, :, None, :]
        sampled = multi_scale_deformable_attn(value, spatial_shapes, level_start_index, locations, weights)
        p = self.dropout if self.training else 0.0
        if p or self.gated or self.branch:
            return self._feed_forward(self._joined(self.norm1, self.output, sampled, queries, p, seed, 0), p, seed)
        x = self.norm1(self.output(sampled, residual=queries), checkpoint=self.checkpoint)
        hidden = self.up(x, activation=self.activation, checkpoint=self.checkpoint)
        return self.norm2(self.down(hidden, residual=x, checkpoint=self.checkpoint), checkpoint=self.checkpoint)


    def _joined(self, norm, product, x, residual, p, seed, place):
        """A block's last product, its dropout, the residual and the norm."""
        if not p and not self.branch:  # the product brings the residual along
            return norm(product(x, residual=residual))
        return norm.join(product(x), residual, dropout=p, seed=seed, sequence=3 * self.index + place)

    def _feed_forward(self, x, p, seed):
        how = {"seed": seed, "sequence": 3 * self.index + 1}
        if self.gated:
            hidden = gated_linear(x, self.up.weight, self.up.bias, activation=self.activation, dropout=p, **how)
        else:
            hidden = self.up(x, activation=self.activation)
            if p:
                hidden = drop(hidden, p, **how)
        return self._joined(self.norm2, self.down, hidden, x, p, seed, 2)


def example_inputs(layer: DeformableEncoderLayer, batch: int, shapes, queries: int | None = None, seed: int = 0):
    """Random queries on the centres of the levels' pixels (or ``queries`` of them anywhere), as a dict of arguments."""
    parameter = layer.value.weight
    device, dtype, width = parameter.device, parameter.dtype, parameter.size(1)
    gen = torch.Generator(device="cpu").manual_seed(seed)
    table = torch.tensor(shapes, dtype=torch.int64)
    sizes = table.prod(-1)
    centres = torch.cat([torch.stack(torch.meshgrid((torch.arange(h) + 0.5) / h, (torch.arange(w) + 0.5) / w,
                                                    indexing="ij")[::-1], -1).view(-1, 2) for h, w in shapes])
    features = torch.randn(batch, int(sizes.sum()), width, generator=gen).to(device, dtype)
    if queries is None:
        x, points = features, centres.expand(batch, -1, 2)
    else:
        x = torch.randn(batch, queries, width, generator=gen).to(device, dtype)
        points = torch.rand(batch, queries, 2, generator=gen)
    return {"queries": x, "features": features,
            "reference_points": points[:, :, None, :].expand(-1, -1, len(shapes), 2).to(device, dtype),
            "spatial_shapes": table.to(device), "level_start_index": (sizes.cumsum(0) - sizes).to(device)}


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--batch", type=int, default=2)
    parser.add_argument("--queries", type=int, default=None, help="decoder-like queries instead of the encoder's own rows")
    parser.add_argument("--dtype", choices=("bfloat16", "float32"), default="bfloat16")
    parser.add_argument("--forward", action="store_true", help="the forward pass alone")
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--dropout", type=float, default=0.0)
    parser.add_argument("--gated", action="store_true", help="a gated feed-forward, of the same width")
    parser.add_argument("--norms", choices=("sum", "branch"), default="sum")
    args = parser.parse_args()
    if not torch.cuda.is_available():
        raise SystemExit("needs a CUDA device")
    plain = not args.dropout and not args.gated and args.norms == "sum"
    for checkpoint in (None, "int8") if plain and not args.forward else (None,):
        torch.manual_seed(0)
        layer = DeformableEncoderLayer(activation="gelu", checkpoint=checkpoint, device="cuda",
                                       dtype=getattr(torch, args.dtype), dropout=args.dropout, gated=args.gated,
                                       norms=args.norms).train(not args.forward)
        inputs = example_inputs(layer, args.batch, cases.DETR_SHAPES, args.queries)
        inputs["seed"] = torch.zeros((), dtype=torch.int64, device="cuda")  # the step's number

        def step():
            if args.forward:
                with torch.no_grad():
                    return layer(**inputs)
            layer.zero_grad(set_to_none=True)
            out = layer(**inputs)
            held = torch.cuda.memory_allocated()
            out.backward(torch.ones_like(out))
            inputs["seed"] += 1
            return held

        before = torch.cuda.memory_allocated()
        for _ in range(3):
            held = step()
        torch.cuda.synchronize()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(args.steps):
            step()
        end.record()
        torch.cuda.synchronize()
        line = f"checkpoint={checkpoint}: {start.elapsed_time(end) / args.steps:.3f} ms a step"
        if not args.forward:
            line += f", {(held - before) / 1e6:.0f} MB held between forward and backward"
        print(line)


if __name__ == "__main__":
    main()
