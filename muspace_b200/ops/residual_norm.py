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
gradients there: with ``return_sum`` at the sum returned (in float16 they are not finite
where it is not). Without it, rows that 16 bits would not hold as a sum, whose mean is
more than four times their spread or which go beyond float16's range, are kept
normalised, and their gradients are those of the sum before any rounding. That of
``norm_add`` takes the input. Masks are made again. Gradients
of weight, bias and gate are added up in an order that does not depend on scheduling.
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
KEEP = 16  # MSDA_NORM_KEEP


# What a call has beside its tensors, as a tuple: branch, kind, residual scale, eps,
# threshold, seed, sequence, groups of the gate, whether the sum is asked for.
#
# Both passes below are written for few Python steps: in training, the host's part of a
# call with short rows takes longer than its kernels.


def _fresh(like: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of the same shape and kind."""
    return torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)


def _forward(module: NativeModule, rule, x, residual, weight, bias, gate, seed_tensor, keep: bool):
    """``(output or None, sum or None, statistics or None)``."""
    branch, kind, scale, eps, threshold, seed, sequence, groups, want_sum = rule
    rows, x_stride = rows_of(x)
    residual, r_stride = rows_of(residual)
    count, width = map(int, rows.shape)  # tensors while tracing
    code = WIDE_DTYPE_CODES[x.dtype]
    param = weight if weight is not None else bias
    gate_code = code
    gate_stride = 0
    if gate is not None:
        gate_code = WIDE_DTYPE_CODES[gate.dtype]
        gate, gate_stride = rows_of(gate)
    out = None if branch else _fresh(x)
    total = _fresh(x) if branch or want_sum or keep else None
    statistics = mean = rstd = None
    if keep:
        statistics = torch.empty((2, count), dtype=torch.float32, device=x.device)
        mean = statistics.data_ptr()
        rstd = mean + 4 * count
        if not branch and not want_sum:  # nobody but the backward pass sees the sum
            kind |= KEEP
    module.plain_call("msda_norm_add_forward" if branch else "msda_add_norm_forward")(x.device, ResidualNormArgs(
        code, code if param is None else WIDE_DTYPE_CODES[param.dtype], gate_code, kind, count, width, groups,
        x_stride, r_stride, gate_stride, 0, 0, 0, scale, eps, threshold, seed, sequence, pointer(seed_tensor),
        rows.data_ptr(), residual.data_ptr(), pointer(gate), pointer(weight), pointer(bias), pointer(out),
        pointer(total), mean, rstd))
    return out, total, statistics


class _ResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, gate, seed_tensor, rule):
        ctx.set_materialize_grads(False)
        needs = ctx.needs_input_grad
        out, total, statistics = _forward(native_module(), rule, x, residual, weight, bias, gate, seed_tensor,
                                          any(needs))
        need_x, _, need_w, need_b, need_gate = needs[:5]
        ctx.rule = rule
        ctx.kinds = (x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype,
                     gate if gate is None else (gate.dtype, gate.shape))
        if rule[0]:
            # the residual's gradient alone needs nothing of the norm
            some = need_x or need_w or need_b or need_gate
            ctx.save_for_backward(x if some else None, weight if need_x or need_gate else None,
                                  bias if need_gate else None, gate, statistics if some else None, seed_tensor, None)
            return total
        ctx.save_for_backward(x if need_gate else None, weight, None, gate, statistics, seed_tensor, total)
        return (out, total) if rule[-1] else out

    @staticmethod
    def backward(ctx, *grads):
        # the wrapper costs 3 us; it is needed where a graph of this pass is asked for
        return _backward_once(ctx, *grads) if torch.is_grad_enabled() else _backward(ctx, *grads)


def _backward(ctx, *grads):
    branch, kind, scale, eps, threshold, seed, sequence, groups, want_sum = rule = ctx.rule
    grad_y, grad_s = (None, grads[0]) if branch else (grads[0], grads[1] if want_sum else None)
    first = grad_s if grad_y is None else grad_y
    if first is None:
        return (None,) * 7
    x, weight, bias, gate, statistics, seed_tensor, total = ctx.saved_tensors
    need_x, need_r, need_w, need_b, need_gate = ctx.needs_input_grad[:5]
    if not branch and grad_y is None:
        need_w = need_b = False
    dx = dr = dw = db = dgate = None
    passed = None  # the residual's gradient where nothing of the norm is in it; dr is the kernel's to write
    same = False
    if branch:
        if need_r and (scale == 1.0 or not (need_x or need_w or need_b or need_gate)):
            passed, need_r = grad_s if scale == 1.0 else grad_s * scale, False
    elif need_x and need_r:
        # without gate and dropout both parts of the sum have one gradient
        same = scale == 1.0 and gate is None and threshold == 0
    if not (need_x or need_r or need_w or need_b or need_gate):
        return None, passed, None, None, None, None, None
    param, gate_kind = ctx.kinds
    device, dtype = first.device, first.dtype
    code = WIDE_DTYPE_CODES[dtype]
    rows, stride = rows_of(first)
    count, width = map(int, rows.shape)
    y_stride = s_stride = x_stride = total_stride = gate_stride = 0
    y_at = s_at = total_at = mean = rstd = None
    if grad_y is not None:
        y_at, y_stride = rows.data_ptr(), stride
        if grad_s is not None and (need_x or need_r or need_gate):  # what reaches the sum reaches no weight or bias
            more, s_stride = rows_of(grad_s)
            s_at = more.data_ptr()
    else:
        s_at, s_stride = rows.data_ptr(), stride
    if x is not None:
        x, x_stride = rows_of(x)
    if total is not None:
        total_at, total_stride = total.data_ptr(), width  # laid out by the forward
    gate_code = code
    if gate_kind is not None:
        gate_code = WIDE_DTYPE_CODES[gate_kind[0]]
        gate, gate_stride = rows_of(gate)
    if statistics is not None:
        mean = statistics.data_ptr()
        rstd = mean + 4 * count
    if need_x:
        dx = _fresh(first)
    if need_r and not same:
        dr = _fresh(first)
    if need_w:
        dw = torch.empty(width, dtype=param, device=device)
    if need_b:
        db = torch.empty(width, dtype=param, device=device)
    if need_gate:
        dgate = torch.empty(gate_kind[1], dtype=gate_kind[0], device=device)
    native_module().plain_call("msda_norm_add_backward" if branch else "msda_add_norm_backward")(
        device, ResidualNormArgs(
            code, WIDE_DTYPE_CODES[param], gate_code, kind, count, width, groups, x_stride, 0, gate_stride,
            total_stride, y_stride, s_stride, scale, eps, threshold, seed, sequence, pointer(seed_tensor), pointer(x),
            None, pointer(gate), pointer(weight), pointer(bias), None, total_at, mean, rstd, y_at, s_at, pointer(dx),
            pointer(dr), pointer(dw), pointer(db), pointer(dgate)))
    return dx, dx if same else passed if dr is None else dr, dw, db, dgate, None, None


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
    if len(own) == len(shape) and own[-1] == shape[-1]:
        upto = len(lead)
        while upto and own[upto - 1] == 1:
            upto -= 1
        if own[:upto] == tuple(lead[:upto]):
            return gate if gate.dim() else gate.reshape(1), int(prod(lead[:upto]))  # tensors while tracing
    return _expanded("gate", gate.float(), shape), int(prod(lead))


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
    rule = (operator == "norm_add", KINDS[kind], float(residual_scale), float(eps), threshold, number, sequence, groups,
            want_sum)
    tensors = (input, residual, weight, bias, gate)
    try:
        if autograd_sees(*tensors):
            output = _ResidualNormFunction.apply(*tensors, seed_tensor, rule)
        else:
            out, total, _ = _forward(module, rule, *tensors, seed_tensor, False)
            output = total if rule[0] else (out, total) if want_sum else out
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
    in ``dropout``. The norm is taken of the sum before it is rounded to its dtype; with
    ``return_sum`` the gradients are those at the sum as it is returned.
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
