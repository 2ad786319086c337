"""Gated feed-forward product: both projections, the activation, their product and
dropout in one kernel, forward and backward.

``y = D(act(x Wg^T + bg) * (x Wu^T + bu))``; the weight holds ``Wg`` above ``Wu``, so
both products are one, and what it is made of never reaches memory in inference. In
training the forward keeps the factors ``P = D'(act'(zg) zu)`` and ``Q = D'(act(zg))``
(``D'`` multiplies as ``D`` does): two numbers per output element, as many as ``zg`` and
``zu`` would be, and the mask is in them. Beside bfloat16 they are float16, each eight
neighbours under an exponent of their own (11 bits down to 2^-28 of the largest of the eight;
smaller ones are off by up to 2^-39 of it).

Backward: ``dz = [g P, g Q]``, ``dx = dz W``, ``dW = dz^T x``, ``db`` the sum of ``dz``
over rows; ``dz`` of a dropped element is 0, whatever ``g``. In
bfloat16 ``dz`` is rounded to bfloat16 before the two products, as a tensor core takes
it. Forward and backward, kernels alone, on a B200: 40000 x 256 x 512 bfloat16 gelu
with dropout 171 us, 22223 x 256 x 512 float32 silu 338; forward of one row, 4096 x
4096 bfloat16, 13.5.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ..runtime.kernel_dispatch import record_dispatch_report
from ..runtime.native import GatedLinearArgs, NativeModule
from ._layer_common import DTYPE_CODES, autograd_sees, check_tensor, decide, failed, native_module, pointer, rows_of
from .dropout import check_rule
from .linear_act import ACTIVATIONS

OPERATOR_NAME = "gated_linear"


def _forward(module: NativeModule, x, weight, bias, seed_tensor, activation: str, rule, keep: bool):
    """``(output, factors)``; every tensor float32 or bfloat16."""
    rows, x_stride = rows_of(x)
    weight, w_stride = rows_of(weight)
    count, features, width = rows.size(0), weight.size(1), weight.size(0) // 2
    out = x.new_empty((*x.shape[:-1], width))
    factors = exponents = None
    if keep and x.dtype == torch.bfloat16:  # halves, and behind them the bytes
        factors = torch.empty(4 * count * width + 8 * count * -(-width // 32), dtype=torch.uint8, device=x.device)
        exponents = factors.data_ptr() + 4 * count * width
    elif keep:
        factors = x.new_empty((count, 2 * width))
    if bias is not None:
        bias = bias.contiguous()
    args = GatedLinearArgs(DTYPE_CODES[x.dtype], ACTIVATIONS[activation], count, features, width, x_stride, w_stride,
                           width, 0, *rule, pointer(seed_tensor), rows.data_ptr(), weight.data_ptr(), pointer(bias),
                           out.data_ptr(), pointer(factors), exponents)
    module.plain_call("msda_gated_linear_forward")(x.device, args)
    return out, factors


class _GatedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, seed_tensor, activation, rule):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        out, factors = _forward(native_module(), x, weight, bias, seed_tensor, activation, rule,
                                need_x or need_w or need_b)
        ctx.save_for_backward(x if need_w else None, weight if need_x else None, factors)
        ctx.sizes = (x.shape, weight.shape)
        return out

    @staticmethod
    def backward(ctx, grad):
        # the wrapper costs 3 us; it is needed where a graph of this pass is asked for
        return _backward_once(ctx, grad) if torch.is_grad_enabled() else _backward(ctx, grad)


def _backward(ctx, grad):
    x, weight, factors = ctx.saved_tensors
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    x_shape, w_shape = ctx.sizes
    g, g_stride = rows_of(grad)
    dx = grad.new_empty(x_shape) if need_x else None
    dw = grad.new_empty(w_shape) if need_w else None
    db = grad.new_empty(w_shape[:1]) if need_b else None
    x_stride = w_stride = 0
    if x is not None:
        x, x_stride = rows_of(x)
    if weight is not None:
        weight, w_stride = rows_of(weight)
    count, width = g.shape
    exponents = factors.data_ptr() + 4 * count * width if grad.dtype == torch.bfloat16 else None
    args = GatedLinearArgs(DTYPE_CODES[grad.dtype], 0, count, w_shape[1], width, x_stride, w_stride, 0, g_stride, 0, 0,
                           0, None, pointer(x), pointer(weight), None, None, factors.data_ptr(), exponents,
                           g.data_ptr(), pointer(dx), pointer(dw), pointer(db))
    native_module().plain_call("msda_gated_linear_backward")(grad.device, args)
    return dx, dw, db, None, None, None


_backward_once = once_differentiable(_backward)


def gated_linear(input: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 activation: str = "silu", dropout: float = 0.0, seed=None, sequence: int = 0,
                 backend: str = "auto") -> torch.Tensor:
    """``dropout(act(input @ gate.T + gate_bias) * (input @ up.T + up_bias))`` (differentiable).

    input ``(..., in)``; weight ``(2 * out, in)``, the gate's rows before up's; bias ``(2 *
    out,)`` in the same order, or None; activation ``"none"``, ``"relu"``, ``"gelu"`` (by the
    normal distribution function) or ``"silu"``, of the gate. All of one dtype: bfloat16,
    float32 (24-bit products), or float16, which runs as float32. ``dropout``, ``seed`` and
    ``sequence`` as in ``dropout``, on the output ``(..., out)``.
    """
    check_tensor(input, "input")
    check_tensor(weight, "weight", input)
    if bias is not None:
        check_tensor(bias, "bias", input)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if input.dim() == 0 or weight.dim() != 2:
        raise ValueError("input must have at least one dimension and weight two")
    both, in_features = weight.shape
    if both % 2:
        raise ValueError(f"weight must have an even number of rows, the gate's and up's, got {both}")
    if input.size(-1) != in_features:
        raise ValueError(f"input has {input.size(-1)} features, weight takes {in_features}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must have shape ({both},), got {tuple(bias.shape)}")
    *rule, seed_tensor = check_rule(dropout, seed, sequence)
    module, report = decide(OPERATOR_NAME, backend, input, weight, bias, seed_tensor)
    dtype = input.dtype
    if dtype == torch.float16:
        input, weight, bias = (t if t is None else t.float() for t in (input, weight, bias))
    try:
        if autograd_sees(input, weight, bias):
            output = _GatedLinearFunction.apply(input, weight, bias, seed_tensor, activation, rule)
        else:
            output, _ = _forward(module, input, weight, bias, seed_tensor, activation, rule, False)
    except RuntimeError as exc:
        failed(report, str(exc))
        raise
    record_dispatch_report(report)
    return output if dtype != torch.float16 else output.to(dtype)


__all__ = ["gated_linear"]
