"""Norms fused with the residual they belong to, its gate, its scale and dropout,
forward and backward.

``add_norm`` joins a block's output to the residual stream and normalises the sum:
``s = residual_scale * residual + gate * D(input)``, ``y = norm(s)``; the sum goes on
as the stream of a pre-norm layer. ``norm_add`` normalises the block's output before
it joins: ``s = residual_scale * residual + gate * D(norm(input))``. Each reads its
rows once and writes each result once. ``norm`` is a layer norm or, without the mean,
a root-mean-square norm; ``D`` is ``dropout``, with the same mask for the same seed,
sequence, rows and columns.

The backward pass of ``add_norm`` takes the sum as it was stored, and gives the
gradients there; that of ``norm_add`` takes the input. Masks are made again. Gradients of weight, bias and gate are
added up in an order that does not depend on scheduling.
"""

from __future__ import annotations

from math import prod

import torch
from torch.autograd.function import once_differentiable

from ..runtime.kernel_dispatch import record_dispatch_report
from ..runtime.native import NativeModule, ResidualNormArgs
from ._layer_common import WIDE_DTYPE_CODES, autograd_sees, check_tensor, decide, failed, native_module, pointer, rows_of
from .dropout import check_rule

KINDS = {"layer": 0, "rms": 1}


class _Rule:
    """What a call has beside its tensors."""

    __slots__ = ("branch", "kind", "scale", "eps", "threshold", "seed", "sequence", "groups", "want_sum")

    def __init__(self, branch, kind, scale, eps, threshold, seed, sequence, groups, want_sum):
        self.branch, self.kind, self.scale, self.eps = branch, kind, scale, eps
        self.threshold, self.seed, self.sequence = threshold, seed, sequence
        self.groups, self.want_sum = groups, want_sum


def _args(rule: _Rule, dtype, weight, bias, gate, count: int, width: int, seed_tensor) -> ResidualNormArgs:
    code = WIDE_DTYPE_CODES[dtype]
    kind = weight if weight is not None else bias
    args = ResidualNormArgs(code, code if kind is None else WIDE_DTYPE_CODES[kind.dtype],
                            code if gate is None else WIDE_DTYPE_CODES[gate.dtype], rule.kind, count, width,
                            rule.groups)
    args.residual_scale, args.eps = rule.scale, rule.eps
    args.threshold, args.seed, args.sequence = rule.threshold, rule.seed, rule.sequence
    args.seed_at = pointer(seed_tensor)
    args.weight, args.bias = pointer(weight), pointer(bias)
    return args


def _gate_rows(args, gate, width: int):
    """Lays the gate out as rows, one to a group, and notes them; the tensor to hold."""
    if gate is not None:
        gate, args.gate_stride = rows_of(gate)
        args.gate = gate.data_ptr()
    return gate


def _forward(module: NativeModule, rule: _Rule, x, residual, weight, bias, gate, seed_tensor, keep: bool):
    """``(output or None, sum or None, statistics or None)``."""
    rows, x_stride = rows_of(x)
    residual, r_stride = rows_of(residual)
    count, width = map(int, rows.shape)  # tensors while tracing
    args = _args(rule, x.dtype, weight, bias, gate, count, width, seed_tensor)
    gate = _gate_rows(args, gate, width)
    args.input, args.input_stride = rows.data_ptr(), x_stride
    args.residual, args.residual_stride = residual.data_ptr(), r_stride
    out = total = statistics = None
    if not rule.branch:
        out = x.new_empty(x.shape)
        args.output = out.data_ptr()
    if rule.branch or rule.want_sum or keep:
        total = x.new_empty(x.shape)
        args.sum = total.data_ptr()
    if keep:
        statistics = torch.empty((2 - rule.kind, count), dtype=torch.float32, device=x.device)
        args.rstd = statistics.data_ptr()
        if rule.kind == 0:
            args.mean = args.rstd + 4 * count if count else args.rstd
    module.plain_call("msda_norm_add_forward" if rule.branch else "msda_add_norm_forward")(x.device, args)
    return out, total, statistics


class _ResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, gate, seed_tensor, rule):
        ctx.set_materialize_grads(False)
        keep = any(ctx.needs_input_grad)
        out, total, statistics = _forward(native_module(), rule, x, residual, weight, bias, gate, seed_tensor, keep)
        need_x, need_r, need_w, need_b, need_gate = ctx.needs_input_grad[:5]
        if rule.branch:
            # the residual's gradient alone needs nothing of the norm
            some = need_x or need_w or need_b or need_gate
            kept = (x if some else None, weight if need_x or need_gate else None, bias if need_gate else None,
                    gate, statistics if some else None, seed_tensor)
        else:
            kept = (x if need_gate else None, weight, None, gate, statistics, seed_tensor)
        ctx.rule = rule
        ctx.width = x.size(-1)
        ctx.kinds = (x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype,
                     gate if gate is None else (gate.dtype, gate.shape))
        ctx.save_for_backward(*kept, None if rule.branch else total)
        if rule.branch:
            return total
        return (out, total) if rule.want_sum else out

    @staticmethod
    def backward(ctx, *grads):
        # the wrapper costs 3 us; it is needed where a graph of this pass is asked for
        return _backward_once(ctx, *grads) if torch.is_grad_enabled() else _backward(ctx, *grads)


def _backward(ctx, *grads):
    rule = ctx.rule
    grad_y, grad_s = (None, grads[0]) if rule.branch else (grads[0], grads[1] if rule.want_sum else None)
    first = grad_s if grad_y is None else grad_y
    if first is None:
        return (None,) * 7
    x, weight, bias, gate, statistics, seed_tensor, total = ctx.saved_tensors
    need_x, need_r, need_w, need_b, need_gate = ctx.needs_input_grad[:5]
    normed = rule.branch or grad_y is not None
    need_w, need_b = need_w and normed, need_b and normed
    shape, width = first.shape, ctx.width
    plain = rule.scale == 1.0
    dx = dr = dw = db = dgate = None
    if rule.branch:
        if need_r and (plain or not (need_x or need_w or need_b or need_gate)):
            dr, need_r = grad_s if plain else grad_s * rule.scale, False  # nothing of the norm is in it
        same = False
    else:
        # without gate and dropout both parts of the sum have one gradient
        same = need_x and need_r and plain and gate is None and rule.threshold == 0
    if not (need_x or need_r or need_w or need_b or need_gate):
        return None, dr, None, None, None, None, None
    kind, gate_kind = ctx.kinds
    count = first.numel() // width if width else prod(shape[:-1])
    args = _args(rule, first.dtype, weight, bias, gate, count, width, seed_tensor)
    args.weight_dtype = WIDE_DTYPE_CODES[kind]
    gate = _gate_rows(args, gate, width)
    hold = []
    if grad_y is not None:
        g, args.grad_output_stride = rows_of(grad_y)
        args.grad_output = g.data_ptr()
        hold.append(g)
    if grad_s is not None:
        g, args.grad_sum_stride = rows_of(grad_s)
        args.grad_sum = g.data_ptr()
        hold.append(g)
    if x is not None:
        x, args.input_stride = rows_of(x)
        args.input = x.data_ptr()
    if total is not None:
        total, args.sum_stride = rows_of(total)
        args.sum = total.data_ptr()
    if statistics is not None:
        args.rstd = statistics.data_ptr()
        if rule.kind == 0:
            args.mean = args.rstd + 4 * count if count else args.rstd
    if need_x:
        dx = first.new_empty(shape)
        args.grad_input = dx.data_ptr()
    if need_r and not same:
        dr = first.new_empty(shape)
        args.grad_residual = dr.data_ptr()
    if need_w:
        dw = torch.empty(width, dtype=kind, device=first.device)
        args.grad_weight = dw.data_ptr()
    if need_b:
        db = torch.empty(width, dtype=kind, device=first.device)
        args.grad_bias = db.data_ptr()
    if need_gate:
        dgate = torch.empty(gate_kind[1], dtype=gate_kind[0], device=first.device)
        args.grad_gate = dgate.data_ptr()
    if not rule.branch and not (need_x or need_r or need_gate):
        args.grad_sum = None  # what reaches the sum does not reach weight and bias
    native_module().plain_call("msda_norm_add_backward" if rule.branch else "msda_add_norm_backward")(
        first.device, args)
    return dx, dx if same else dr, dw, db, dgate, None, None


_backward_once = once_differentiable(_backward)


def _check(name: str, tensor, input: torch.Tensor) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if tensor.dtype not in (input.dtype, torch.float32):
        raise TypeError(f"{name} must have the dtype of input ({input.dtype}) or float32")


def _expanded(name: str, tensor: torch.Tensor, shape) -> torch.Tensor:
    try:
        return tensor.expand(shape)
    except RuntimeError as exc:
        raise ValueError(f"{name} {tuple(tensor.shape)} cannot be broadcast to {tuple(shape)}") from exc


def _groups_of(gate: torch.Tensor, shape) -> tuple[torch.Tensor, int]:
    """The gate, and how many rows it has: neighbouring rows share one where its
    leading dimensions are those of ``shape`` up to some place and 1 from there on.
    A gate of any other shape is broadcast to a row for each, in float32, so that the
    gradients that are then summed to its own shape are not rounded before."""
    lead = shape[:-1]
    own = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape)
    if own[-1] == shape[-1]:
        upto = len(lead)
        while upto and own[upto - 1] == 1:
            upto -= 1
        if own[:upto] == tuple(lead[:upto]):
            return gate, prod(lead[:upto])
    return _expanded("gate", gate.float(), shape), prod(lead)


def _call(operator: str, input, residual, weight, bias, gate, residual_scale, kind, eps, p, seed, sequence, want_sum,
          backend):
    check_tensor(input, "input")
    check_tensor(residual, "residual", input)
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {sorted(KINDS)}, got {kind!r}")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    for name, tensor in (("weight", weight), ("bias", bias)):
        if tensor is None:
            continue
        _check(name, tensor, input)
        if tensor.shape != input.shape[-1:]:
            raise ValueError(f"{name} must have shape ({input.size(-1)},), got {tuple(tensor.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one dtype")
    threshold, number, sequence, seed_tensor = check_rule(p, seed, sequence)
    if residual.shape != input.shape:
        residual = _expanded("residual", residual, input.shape)
    groups = 1
    if gate is not None:
        _check("gate", gate, input)
        gate, groups = _groups_of(gate, input.shape)
    module, report = decide(operator, backend, input, residual, weight, bias, gate, seed_tensor)
    weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
    rule = _Rule(operator == "norm_add", KINDS[kind], float(residual_scale), float(eps), threshold, number, sequence,
                 groups, want_sum)
    tensors = (input, residual, weight, bias, gate)
    try:
        if autograd_sees(*tensors):
            output = _ResidualNormFunction.apply(*tensors, seed_tensor, rule)
        else:
            out, total, _ = _forward(module, rule, *tensors, seed_tensor, False)
            output = total if rule.branch else (out, total) if want_sum else out
    except RuntimeError as exc:
        failed(report, str(exc))
        raise
    record_dispatch_report(report)
    return output


def add_norm(input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
             bias: torch.Tensor | None = None, *, gate: torch.Tensor | None = None, residual_scale: float = 1.0,
             kind: str = "layer", eps: float = 1e-5, dropout: float = 0.0, seed=None, sequence: int = 0,
             return_sum: bool = False, backend: str = "auto"):
    """``norm(s)`` of the sum ``s = residual_scale * residual + gate * dropout(input)``, and with
    ``return_sum`` the pair ``(norm(s), s)`` (differentiable).

    input ``(..., n)`` in bfloat16, float16 or float32; residual broadcastable to it;
    weight and bias ``(n,)`` or None, both of input's dtype or both float32; gate
    broadcastable to input, of its dtype or float32, or None: ``(n,)`` scales channels,
    ``(batch, 1, ..., n)`` those of each sample, and no copy is made of either; kind
    ``"layer"`` (``(s - mean) / sqrt(var + eps) * weight + bias``) or ``"rms"`` (``s /
    sqrt(mean(s^2) + eps) * weight + bias``). ``dropout``, ``seed`` and ``sequence`` as
    in ``dropout``. The norm is taken of the sum before it is rounded to its dtype.
    """
    return _call("add_norm", input, residual, weight, bias, gate, residual_scale, kind, eps, dropout, seed, sequence,
                 bool(return_sum), backend)


def norm_add(input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
             bias: torch.Tensor | None = None, *, gate: torch.Tensor | None = None, residual_scale: float = 1.0,
             kind: str = "layer", eps: float = 1e-5, dropout: float = 0.0, seed=None, sequence: int = 0,
             backend: str = "auto") -> torch.Tensor:
    """``residual_scale * residual + gate * dropout(norm(input))`` (differentiable).

    Arguments as in ``add_norm``; the norm is that of the input.
    """
    return _call("norm_add", input, residual, weight, bias, gate, residual_scale, kind, eps, dropout, seed, sequence,
                 False, backend)


__all__ = ["add_norm", "norm_add"]
